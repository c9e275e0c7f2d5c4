// Matrix product in 8-bit integers with a scale for each token (row of x) and each channel (row of W), and the rounding of rows to 8 bits.
//
//   y[m][n] = act( (sum_k xq[m][k] wq[n][k]) * sx[m] * sw[n] + bias[n] )        xq, wq in -128 .. 127, sums exact in int32
//   row -> codes: s = amax * (1 / 127), q = rint(x * (127 / amax)), amax = max(max |x|, 2^-119)
//
// The sums are v_mfma_i32_16x16x64_i8 and v_mfma_i32_32x32x32_i8: 16 bytes a lane and operand, row (lane & 15) or (lane & 31), a run of 16 k
// for each lane further on. The order of k inside an instruction is the same for both operands, so it does not matter; W is the first
// operand, so that a lane's results are neighbouring channels of one token.
// W is packed: rows padded with zeros to 64 bytes (or a multiple of 128), cut into blocks of 16 rows x 64 bytes, a kilobyte
// each, in which bytes 16 q .. 16 q + 15 of row t are the 16 bytes at 256 q + 16 t: what lane (t, q) of the first instruction takes. A
// wavefront's load of an operand is then one kilobyte side by side. Few tokens are packed too; many stay rows, of which the tiles read 64
// bytes at a time (rounding 8192 rows of 8192 straight into packed blocks takes 89 us, pieces of 16 bytes scattered by different
// workgroups; into rows 32 to 34). 29 tokens x 10240 x 5120: both operands as rows, 16 pieces of 64 bytes a load, 31 us; packed 13.
// Epilogue in fp32, one rounding per operation, one to the type of y.
#include "hrf_common.h"
#include <algorithm>
#include <type_traits>

enum { I8_F32 = 0, I8_F16 = 1, I8_BF16 = 2, I8_INT8 = 3 };

typedef int i8_v4 __attribute__((ext_vector_type(4)));
#define I8_GLOBAL __attribute__((address_space(1)))
#define I8_LDS __attribute__((address_space(3)))

template <int K> struct I8Type;
template <> struct I8Type<I8_F32> { typedef float T; static __device__ float up(float x) { return x; } static __device__ float down(float x) { return x; } };
template <> struct I8Type<I8_F16> { typedef __half T; static __device__ float up(__half x) { return __half2float(x); } static __device__ __half down(float x) { return __float2half_rn(x); } };
template <> struct I8Type<I8_BF16> { typedef __bf16 T; static __device__ float up(__bf16 x) { return (float)x; } static __device__ __bf16 down(float x) { return (__bf16)x; } };

// ------------------------------------------------------------------------------------------------ rows -> codes and scales
// 16 bytes of a row, at any address (unaligned accesses are the hardware's).
template <int K> struct I8Piece { static constexpr int n = 16 / (int)sizeof(typename I8Type<K>::T); typename I8Type<K>::T v[16 / sizeof(typename I8Type<K>::T)]; };

template <int K>
__device__ __forceinline__ void i8_get(I8Piece<K>& v, const typename I8Type<K>::T* from) { __builtin_memcpy(&v, from, 16); }

__device__ __forceinline__ uint32_t i8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }     // |x| as an integer: the order of the values, NaN on top

// amax -> factor of the codes and stored scale. A row that is not finite gets a scale that is not, and codes 0: its outputs are NaN.
__device__ __forceinline__ float i8_factor(uint32_t top, float& scale)
{
    const float amax = __uint_as_float(max(top, 0x04000000u));      // 2^-119: 127 / amax stays finite, a row of zeros gives zeros
    scale = amax * (1.0f / 127.0f);
    return top < 0x7f800000u ? 127.0f / amax : 0.0f;
}

// Four values -> four codes in one word. |x| * factor is below 127.0001 (and 0 * NaN converts to 0), so that no clamp is needed.
__device__ __forceinline__ uint32_t i8_code(float x, float factor, bool finite) { return finite ? (uint32_t)(int)rintf(x * factor) & 0xffu : 0u; }

// A launch has fewer than 2^32 threads along an axis: past 2^22 workgroups they are counted along the second one too.
#define I8_GRID_X (1 << 22)
static dim3 i8_grid(int64_t blocks)
{
    return blocks <= I8_GRID_X ? dim3((unsigned)blocks) : dim3(I8_GRID_X, (unsigned)((blocks + I8_GRID_X - 1) / I8_GRID_X));
}
__device__ __forceinline__ int64_t i8_block() { return (int64_t)blockIdx.y * I8_GRID_X + blockIdx.x; }

// Where code k of a row goes. Packed: see above. Otherwise rows of `ld` codes.
template <bool kPacked>
__device__ __forceinline__ int64_t i8_at(int64_t row, int k, int64_t ld)
{
    return kPacked ? ((row >> 4) * (ld >> 6) + (k >> 6)) * 1024 + ((k >> 4) & 3) * 256 + (row & 15) * 16 + (k & 15) : row * ld + k;
}

// kGroup lanes a row (a power of two up to a wavefront, or the whole workgroup of 256 joined through LDS). The row is read once, in 16-byte
// pieces, and stays in registers, kPieces of them a lane. 8192 rows of 8192 bf16: 118 us read twice value by value, 32 us this way
// over and over on one input, 34 on six in turn, 40 to 47 between products.
template <int K, bool kPacked, int kGroup, int kPieces>
__global__ __launch_bounds__(256) void k_quantize_rows(const typename I8Type<K>::T* __restrict__ x, int64_t rows, int cols, int64_t ldx,
                                                            int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale)
{
    __shared__ uint32_t s_max[4];
    constexpr int n = I8Piece<K>::n, kRows = 256 / kGroup;
    const int lane = threadIdx.x % kGroup;
    const int64_t row = i8_block() * kRows + threadIdx.x / kGroup;
    const bool here = row < rows;
    const typename I8Type<K>::T* const from = x + (here ? row : rows - 1) * ldx;
    I8Piece<K> v[kPieces];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        const int k0 = (p * kGroup + lane) * n;
        if (k0 + n <= cols) i8_get<K>(v[p], from + k0);
        else {
#pragma unroll
            for (int k = 0; k < n; ++k) v[p].v[k] = k0 + k < cols ? from[k0 + k] : I8Type<K>::down(0.0f);
        }
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
        for (int k = 0; k < n; ++k) top = max(top, i8_bits(I8Type<K>::up(v[p].v[k])));
#pragma unroll
    for (int s = (kGroup < 64 ? kGroup : 64) / 2; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if (kGroup == 256) {
        if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    }
    if (!here) return;
    float sc;
    const float factor = i8_factor(top, sc);
    const bool finite = top < 0x7f800000u;
    if (lane == 0) scale[row] = sc;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        const int k0 = (p * kGroup + lane) * n;
        if (k0 >= ldq) continue;        // (ldq is a multiple of 8: whole pieces)
        uint32_t word[n / 4];
#pragma unroll
        for (int w = 0; w < n / 4; ++w) {
            word[w] = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) word[w] |= i8_code(I8Type<K>::up(v[p].v[4 * w + k]), factor, finite) << (8 * k);
        }
        int8_t* const to = q + i8_at<kPacked>(row, k0, ldq);
        if (n == 8) *(uint2*)to = make_uint2(word[0], word[n / 4 - 1]);
        else *(uint32_t*)to = word[0];
    }
}

// Rows too long for the registers: read twice, the second time from the cache. Also codes at any address.
template <int K, bool kPacked>
__global__ __launch_bounds__(256) void k_quantize_rows_long(const typename I8Type<K>::T* __restrict__ x, int64_t rows, int cols, int64_t ldx,
                                                            int8_t* __restrict__ q, int ldq, float* __restrict__ scale)
{
    __shared__ uint32_t s_max[4];
    constexpr int n = I8Piece<K>::n;
    const int64_t row = i8_block();
    if (row >= rows) return;
    const typename I8Type<K>::T* const from = x + row * ldx;
    auto get = [&](int k0, I8Piece<K>& v) {
        if (k0 + n <= cols) i8_get<K>(v, from + k0);
        else {
#pragma unroll
            for (int k = 0; k < n; ++k) v.v[k] = k0 + k < cols ? from[k0 + k] : I8Type<K>::down(0.0f);
        }
    };
    uint32_t top = 0;
    for (int k0 = threadIdx.x * n; k0 < cols; k0 += 256 * n) {
        I8Piece<K> v;
        get(k0, v);
#pragma unroll
        for (int k = 0; k < n; ++k) top = max(top, i8_bits(I8Type<K>::up(v.v[k])));
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    float sc;
    const float factor = i8_factor(top, sc);
    const bool finite = top < 0x7f800000u;
    if (threadIdx.x == 0) scale[row] = sc;
    for (int k0 = threadIdx.x * n; k0 < ldq; k0 += 256 * n) {
        I8Piece<K> v;
        get(k0, v);
        int8_t* const to = q + i8_at<kPacked>(row, k0, ldq);
        int8_t code[n];
#pragma unroll
        for (int k = 0; k < n; ++k) code[k] = (int8_t)i8_code(I8Type<K>::up(v.v[k]), factor, finite);
        if (k0 + n <= ldq) __builtin_memcpy(to, code, n);
        else {
#pragma unroll
            for (int k = 0; k < n; ++k)
                if (k0 + k < ldq) to[k] = code[k];
        }
    }
}

// Rows of codes -> rows padded with zeros to ldq, a multiple of 16 bytes.
__global__ __launch_bounds__(256) void k_pad_rows(const int8_t* __restrict__ x, int64_t rows, int cols, int64_t ldx, int8_t* __restrict__ q, int ldq)
{
    const int64_t row = i8_block();
    if (row >= rows) return;
    x += row * ldx;
    q += row * ldq;
    for (int k0 = threadIdx.x * 16; k0 < ldq; k0 += 4096) {
        i8_v4 v = {0, 0, 0, 0};
        if (k0 + 16 <= cols) __builtin_memcpy(&v, x + k0, 16);
        else
            for (int k = 0; k0 + k < cols; ++k) v[k >> 2] |= (int)((uint32_t)(uint8_t)x[k0 + k] << (8 * (k & 3)));
        *(i8_v4*)(q + k0) = v;
    }
}

// Rows of codes -> packed, a thread for each 16 bytes of the result; rows up to the next multiple of 16 are zeros.
__global__ __launch_bounds__(256) void k_pack_rows(const int8_t* __restrict__ x, int64_t rows, int cols, int64_t ldx,
                                                   int8_t* __restrict__ packed, int64_t padded, int64_t pieces)
{
    const int64_t piece = i8_block() * 256 + threadIdx.x;
    if (piece >= pieces) return;
    const int64_t block = piece >> 6, runs = padded >> 6, row = block / runs * 16 + (piece & 15);
    const int k0 = (int)(block % runs) * 64 + ((int)(piece >> 4) & 3) * 16;
    i8_v4 v = {0, 0, 0, 0};
    if (row < rows) {
        const int8_t* from = x + row * ldx + k0;
        if (k0 + 16 <= cols) __builtin_memcpy(&v, from, 16);
        else {
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k0 + 4 * w + k < cols) v[w] |= (int)((uint32_t)(uint8_t)from[4 * w + k] << (8 * k));
        }
    }
    ((i8_v4*)packed)[piece] = v;
}

// ------------------------------------------------------------------------------------------------ product
struct I8Args {
    const int8_t* x;            // codes: packed for few tokens, else rows of ldx bytes
    int64_t ldx;
    const int8_t* w;            // packed
    const float* sx;
    const float* sw;
    const float* bias;
    void* y;
    int64_t ldy;
    int rows, cols, inner;      // inner: padded
    int relu;
};

// acc sx sw, two roundings. The product of two scales of 2^-63 to 2^63 is a normal number. Of others (kWide) the significands are
// multiplied and the exponents put back at the end, so that nothing overflows or loses bits unless the result does. Both give the same bits
// where the first is right; a workgroup takes the second way if one of its scales asks for it. Looking takes 0.4 us of 26 for
// 1021 x 4099 x 2051 and 0.3 of 20.7 for 320000 x 64 x 64.
// 0, inf and NaN are not wide: both ways give the same.
__device__ __forceinline__ bool i8_is_wide(float scale)
{
    const uint32_t bits = i8_bits(scale);
    return bits - 1u < 0x1fffffffu || bits - 0x5f000001u < 0x207fffffu;
}

template <bool kWide>
__device__ __forceinline__ float i8_scaled(int acc, float sx, float sw)
{
    if (!kWide) return (float)acc * (sx * sw);
    asm volatile("" : "+v"(sx), "+v"(sw));      // (the compiler would take all scales apart before it looks, and hold on to the parts)
    return ldexpf((float)acc * (__builtin_amdgcn_frexp_mantf(sx) * __builtin_amdgcn_frexp_mantf(sw)),
                  __builtin_amdgcn_frexp_expf(sx) + __builtin_amdgcn_frexp_expf(sw));
}

template <int K>
__device__ __forceinline__ typename I8Type<K>::T i8_finish(float v, float bias, bool has_bias, bool relu)
{
    if (has_bias) v = v + bias;
    if (relu) v = v < 0.0f ? 0.0f : v;
    return I8Type<K>::down(v);
}

// N neighbouring values, 16 bytes, of a row of y from column n on.
template <typename T, int N>
__device__ __forceinline__ void i8_store(T* row, int n, int cols, bool here, const T* v)
{
    static_assert(N * sizeof(T) == 16, "a piece is 16 bytes");
    if (!here) return;
    if (n + N <= cols) {
        i8_v4 piece;
        __builtin_memcpy(&piece, v, 16);
        asm("" : "+v"(piece));      // (a whole piece: left alone, the last value's store is shared with the other branch)
        __builtin_memcpy(row + n, &piece, 16);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (n + k < cols) row[n + k] = v[k];
    }
}

// 16 bytes from base + offset (each lane its own) to LDS, the wavefront's kilobyte from byte `to` on in the order of its lanes. The
// compiler takes the builtin for this as something every later LDS read may depend on and waits for it at once; here the caller waits
// (s_waitcnt vmcnt, a barrier) before anybody reads. m0 holds the address in LDS; it is an input of the
// statement, so that the compiler writes it and knows.
__device__ __forceinline__ void i8_load_lds(const int8_t* base, uint32_t offset, uint32_t to)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(to), "v"(offset), "s"(base) : "memory");
}

// Block -> tile: the blocks that run on one XCD (every eighth) take neighbouring tiles, in columns of 8 tiles of tokens, so that what they
// read together fits their L2.
__device__ __forceinline__ void i8_tile_of(int tiles_m, int tiles_n, int& tm, int& tn)
{
    const int total = tiles_m * tiles_n, xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
    const int id = xcd * q + min(xcd, r) + (int)(blockIdx.x >> 3);
    const int group = id / (8 * tiles_n), first = group * 8, height = min(8, tiles_m - first), in = id - group * 8 * tiles_n;
    tm = first + in % height;
    tn = in / height;
}

// Tiles of BM = 64 TM tokens x BN = 32 TN WN channels, 2 x WN wavefronts, 32 TM x 32 TN each from v_mfma_i32_32x32x32_i8. A stage is 64 R
// bytes of k in LDS, four stages, filled by direct loads (16 bytes a lane, no registers) three stages ahead. W's packed blocks lie there as
// in memory: 16 lanes that read together read 256 bytes side by side. A token's four 16-byte chunks lie permuted by its number, so that 16
// lanes that read the same chunk of neighbouring tokens hit all 64 banks.
// Everything is dealt out between the products: while the matrix cores work on 32 k, the operands of the next 32 are read from LDS and
// a quarter of the loads of the third stage on is issued (sixteen loads in a row hold the wavefront up for as long as they take
// to issue, half a stage). In the middle of a stage the workgroup meets: the next stage has landed, and nobody reads the one before.
// 8192^3 with 256 x 256 tiles: 456 to 537 us from card to card and run to run (2.05 to 2.4 POP/s; the library's product of the same
// integers reached 2.14 where this one took 469), bound by power: the matrix cores are at work 72 % of the clocks, of which the card makes
// 1.4 to 1.5 GHz under this load (random codes; with zeros a tenth less time). No bank conflicts in LDS. Every 8192 k more take 417 us; the rest are the ends of the four tiles that each CU takes, where nothing is
// multiplied. (Going from tile to tile in one workgroup, the next one's loads on their way meanwhile, took 505 us where one tile a
// workgroup took 483: the registers for that are not there.) 8 wavefronts rather than 4 shorten the ends: 8192 x 8192 x 1024 109 us
// against 119. 128 x 128 tiles read 8.6 GB for the same product in 640 us, 13 TB/s.
template <int K, int TM, int TN, int WN, int R>
__global__ __launch_bounds__(128 * WN, (TM * TN * WN > 8 ? 1 : 2) * WN / 2) void k_linear_i8(const I8Args A)
{
    constexpr int BM = 64 * TM, BN = 32 * TN * WN, kThreads = 128 * WN, kRun = (BM + BN) * 64, kStage = kRun * R;
    constexpr int kPerRun = (BM + BN) / (32 * WN), kLoads = kPerRun * R;       // loads of a wavefront: of 64 bytes of k, of a stage
    static_assert((BM + BN) % (32 * WN) == 0, "every wavefront loads as much");
    constexpr int kOperands = R * (TM + TN), kProducts = R * TM * TN, kGroups = kProducts % 3 == 0 ? 3 : 2, kEarly = (kLoads + 1) / 2;
    typedef typename I8Type<K>::T T;
    typedef int i8_v16 __attribute__((ext_vector_type(16)));
    __shared__ __align__(16) int8_t s_tile[4 * kStage];
    __shared__ float s_sx[BM], s_sw[BN], s_bias[BN];
    __shared__ int s_wide[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    int tm, tn;
    i8_tile_of((A.rows + BM - 1) / BM, (A.cols + BN - 1) / BN, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int steps = A.inner / (64 * R);

    // Load j of 64 bytes of k is number wave * kPerRun + j of the tile: first the tokens, 16 a load, this lane's row lane / 4 of them (past the
    // end: the last one), its chunk permuted; then the channels, a block of 16 (past the end: the last one).
    uint32_t from[kPerRun];
#pragma unroll
    for (int j = 0; j < kPerRun; ++j) {
        const int sixteen = wave * kPerRun + j;
        from[j] = sixteen < BM / 16 ? (uint32_t)min(sixteen * 16 + (lane >> 2), A.rows - 1 - m0) * (uint32_t)A.ldx + ((lane & 3) ^ (lane >> 4)) * 16
                                    : (uint32_t)(min((n0 >> 4) + sixteen - BM / 16, (A.cols - 1) >> 4) - (n0 >> 4)) * (uint32_t)A.inner * 16 + lane * 16;
    }
    const int8_t* const xb = A.x + (int64_t)m0 * A.ldx;
    const int8_t* const wb = A.w + (int64_t)n0 * A.inner;
    const uint32_t lds = (uint32_t)(uintptr_t)(I8_LDS int8_t*)s_tile + wave * kPerRun * 1024;
    auto load = [&](int i, int s) {
        const int run = i / kPerRun, j = i % kPerRun;
        const int64_t at = (int64_t)min(s, steps - 1) * R + run;
        const bool token = wave * kPerRun + j < BM / 16;
        i8_load_lds((token ? xb : wb) + at * (token ? 64 : 1024), from[j], lds + (s & 3) * kStage + run * kRun + j * 1024);
    };

    i8_v16 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[a][b][k] = 0;
    i8_v4 fr[2][R * (TM + TN)]; // two sets of operands, half a stage each: for every 32 k of the tokens, then of the channels
    const int x_row = (wm * 32 * TM + (lane & 31)) * 64, w_row = (BM / 16 + wn * 2 * TN) * 1024 + ((lane >> 4) & 1) * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
    auto read = [&](int set, int o, int s, int half) {
        const int j = o % (TM + TN), kk = (half * R + o / (TM + TN)) & 1, run = (half * R + o / (TM + TN)) >> 1;
        const int8_t* t = s_tile + (s & 3) * kStage + run * kRun;
        if (j < TM) fr[set][o] = *(const i8_v4*)(t + x_row + ((kk * 2 + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16 + j * 2048);
        else fr[set][o] = *(const i8_v4*)(t + w_row + kk * 512 + (j - TM) * 2048);
    };
    // the products of one set, between them the reads of the other (a half of stage `next`) and half of the loads of stage `ahead`
    auto work = [&](int set, int next, int half, int ahead) {
        const int first = set == 0 ? 0 : kEarly, loads = set == 0 ? kEarly : kLoads - kEarly;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int j = 0; j < kOperands; ++j)
                if (j * kGroups / kOperands == g) read(set ^ 1, j, next, half);
#pragma unroll
            for (int p = g * kProducts / kGroups; p < (g + 1) * kProducts / kGroups; ++p) {
                const int o = p / (TM * TN) * (TM + TN), a = p % (TM * TN) / TM, b = p % TM;
                acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fr[set][o + TM + a], fr[set][o + b], acc[a][b], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kEarly; ++i)
                if (i < loads && i * kGroups / kEarly == g) load(first + i, ahead);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Scales and biases, a thread each, stay in registers until the products are done: nobody waits for them before the first stage.
    static_assert(BM <= kThreads && BN <= kThreads, "a thread for each scale");
    const int tx = min((int)threadIdx.x, BM - 1), tw = min((int)threadIdx.x, BN - 1), nw = min(n0 + tw, A.cols - 1);
    const float scale_x = A.sx[min(m0 + tx, A.rows - 1)], scale_w = A.sw[nw], bias_w = A.bias ? A.bias[nw] : 0.0f;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(i, s);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * kLoads) : "memory");
#pragma unroll
    for (int j = 0; j < R * (TM + TN); ++j) read(0, j, 0, 0);
    for (int s = 0; s < steps; ++s) {
        work(0, s, 1, s + 3);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLoads + kEarly) : "memory");   // stage s + 1 has landed, of two more 3 halves are on their way
        work(1, s + 1, 0, s + 3);       // (past the end: stages that are there, read again and not used)
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // nothing may land in LDS that is somebody else's by then
    s_sx[tx] = scale_x;         // (of the threads past the end the last one's again)
    s_sw[tw] = scale_w;
    s_bias[tw] = bias_w;
    const bool odd = __any(i8_is_wide(scale_x) || i8_is_wide(scale_w));
    if (lane == 0) s_wide[wave] = odd;
    __syncthreads();

    // Epilogue, 32 channels of 32 tokens at a time: a lane holds channels 8 g + 4 (lane / 32) + 0 .. 3 of token lane % 32. For 16-bit y the
    // halves of the wavefront trade, so that a lane has eight neighbouring channels, 16 bytes. (Through LDS, whole rows at a time, this
    // took as long as 2000 k of products: there is no other workgroup on the CU to work meanwhile.)
    const bool has_bias = A.bias != nullptr, relu = A.relu != 0;
    int wide = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) wide |= s_wide[w];
    auto finish = [&](auto kind) {
#pragma unroll
        for (int a = 0; a < TN; ++a) {
            const int nl = wn * 32 * TN + a * 32 + (lane >> 5) * 4;
            float sw[16], bias[16];
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sw[g * 4 + k] = s_sw[nl + g * 8 + k];
                    bias[g * 4 + k] = s_bias[nl + g * 8 + k];
                }
#pragma unroll
            for (int b = 0; b < TM; ++b) {
                const int ml = wm * 32 * TM + b * 32 + (lane & 31), m = m0 + ml;
                const float sx = s_sx[ml];
                T v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = i8_finish<K>(i8_scaled<decltype(kind)::value>(acc[a][b][k], sx, sw[k]), bias[k], has_bias, relu);
                T* const y = (T*)A.y + (int64_t)m * A.ldy;
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) i8_store<T, 4>(y, n0 + nl + g * 8, A.cols, m < A.rows, v + g * 4);
                } else {
#pragma unroll
                    for (int g = 0; g < 4; g += 2) {
                        uint32_t u[4];
                        __builtin_memcpy(u, v + g * 4, 16);         // this lane's four of g, four of g + 1
#pragma unroll
                        for (int h = 0; h < 2; ++h) {               // lower half: all of g, upper half: all of g + 1
                            const auto both = __builtin_amdgcn_permlane32_swap(u[h], u[2 + h], false, false);
                            u[h] = both[0];
                            u[2 + h] = both[1];
                        }
                        T eight[8];
                        __builtin_memcpy(eight, u, 16);
                        i8_store<T, 8>(y, n0 + wn * 32 * TN + a * 32 + (g + (lane >> 5)) * 8, A.cols, m < A.rows, eight);
                    }
                }
            }
            asm volatile("" ::: "memory");      // (one a at a time: the compiler would fetch all the scales first, and spill)
        }
    };
    if (__builtin_amdgcn_readfirstlane(wide) == 0) finish(std::false_type());
    else finish(std::true_type());
}

// Short rows (up to 64 KS values), many of them: bound by the bytes of x and y, so x is rounded on its way in and nothing is written
// between. A wavefront keeps the weights of 64 channels in registers and walks over blocks of 16 tokens; lane (t, q) = (lane & 15, lane >> 4)
// holds 16 values of token t for each 64, finds the row's largest with the three other lanes of the token, and has its operand. The
// channels are dealt to the instructions so that a lane's 16 results are 16 neighbouring channels of one token: 32 bytes of fp16 in a
// row of 128.
struct I8Short {
    const void* x;          // rows as the caller has them
    int64_t ldx;
    const float* sx;        // of integer rows
    int inner;              // not padded
};

template <int X, int K, int KS>
__global__ __launch_bounds__(256) void k_linear_i8_short(const I8Args A, const I8Short B)
{
    typedef typename I8Type<K>::T T;
    const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
    const int waves = (int)gridDim.x * 4, wave = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    const int n0 = (int)blockIdx.y * 64;
    const bool has_bias = A.bias != nullptr, relu = A.relu != 0;
    i8_v4 fw[KS][4];
    float sw[16], bias[16];
    bool odd = false;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        // row a * 4 + t % 4 of the block of 16 that t / 4 names (past the last one: the last again)
        const int64_t block = min((n0 >> 4) + (t >> 2), (A.cols - 1) >> 4);
#pragma unroll
        for (int s = 0; s < KS; ++s) fw[s][a] = *(const i8_v4*)(A.w + (block * KS + s) * 1024 + q * 256 + (a * 4 + (t & 3)) * 16);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int n = min(n0 + q * 16 + k, A.cols - 1);
        sw[k] = A.sw[n];
        odd |= i8_is_wide(sw[k]);
        bias[k] = has_bias ? A.bias[n] : 0.0f;
    }
    const int blocks = (A.rows + 15) / 16;
    for (int blk = wave; blk < blocks; blk += waves) {
        const int m = blk * 16 + t;
        const int64_t row = min(m, A.rows - 1);
        i8_v4 fx[KS];
        float sx;
        if constexpr (X == I8_INT8) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int8_t* const from = (const int8_t*)B.x + row * B.ldx;
                const int k0 = s * 64 + q * 16;
                if (k0 + 16 <= B.inner) __builtin_memcpy(&fx[s], from + k0, 16);
                else {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        fx[s][w] = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k0 + 4 * w + k < B.inner) fx[s][w] |= (int)((uint32_t)(uint8_t)from[k0 + 4 * w + k] << (8 * k));
                    }
                }
            }
            sx = B.sx[row];
        } else {
            typedef typename I8Type<X>::T XT;
            constexpr int n = I8Piece<X>::n, kPieces = 16 / n;
            const XT* const from = (const XT*)B.x + row * B.ldx;
            I8Piece<X> v[KS][kPieces];
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int p = 0; p < kPieces; ++p) {
                    const int k0 = s * 64 + q * 16 + p * n;
                    if (k0 + n <= B.inner) i8_get<X>(v[s][p], from + k0);
                    else {
#pragma unroll
                        for (int k = 0; k < n; ++k) v[s][p].v[k] = k0 + k < B.inner ? from[k0 + k] : I8Type<X>::down(0.0f);
                    }
                }
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int p = 0; p < kPieces; ++p)
#pragma unroll
                    for (int k = 0; k < n; ++k) top = max(top, i8_bits(I8Type<X>::up(v[s][p].v[k])));
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const float factor = i8_factor(top, sx);
            const bool finite = top < 0x7f800000u;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t word = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) word |= i8_code(I8Type<X>::up(v[s][(4 * w + k) / n].v[(4 * w + k) % n]), factor, finite) << (8 * k);
                    fx[s][w] = (int)word;
                }
        }
        __align__(16) T out[16];
        auto finish = [&](auto kind) {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                i8_v4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[s][a], fx[s], acc, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    out[a * 4 + k] = i8_finish<K>(i8_scaled<decltype(kind)::value>(acc[k], sx, sw[a * 4 + k]), bias[a * 4 + k], has_bias, relu);
            }
        };
        if (!__any(odd || i8_is_wide(sx))) finish(std::false_type());
        else finish(std::true_type());
        constexpr int n = 16 / (int)sizeof(T);
#pragma unroll
        for (int p = 0; p < 16 / n; ++p) i8_store<T, n>((T*)A.y + row * A.ldy, n0 + q * 16 + p * n, A.cols, m < A.rows, out + p * n);
    }
}

// Few tokens (up to 16 MT): bound by the bytes of W, which every workgroup reads its part of once: 16 NT channels, the k axis dealt to its
// kWaves wavefronts in runs of 64 bytes, sums joined in LDS. Integer sums: any order gives the same.
template <int K, int MT, int NT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void k_linear_i8_few(const I8Args A)
{
    typedef typename I8Type<K>::T T;
    __shared__ i8_v4 s_part[kWaves][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = (int)blockIdx.x * 16 * NT;
    const int runs = A.inner >> 6, each = (runs + kWaves - 1) / kWaves, begin = wave * each, end = min(begin + each, runs);
    const int8_t* w[NT];
    const int8_t* x[MT];
#pragma unroll
    for (int a = 0; a < NT; ++a) w[a] = A.w + (int64_t)min((n0 >> 4) + a, (A.cols - 1) >> 4) * runs * 1024 + lane * 16;
#pragma unroll
    for (int b = 0; b < MT; ++b) x[b] = A.x + (int64_t)min(b, (A.rows - 1) >> 4) * runs * 1024 + lane * 16;
    i8_v4 acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[a][b] = i8_v4{0, 0, 0, 0};
    constexpr int kAhead = MT * NT > 4 ? 2 : MT * NT > 1 ? 4 : 8;        // runs on their way at a time
    for (int r = begin; r < end; r += kAhead) {
        i8_v4 fw[kAhead][NT], fx[kAhead][MT];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t k = (int64_t)min(r + u, end - 1) * 1024;
#pragma unroll
            for (int a = 0; a < NT; ++a) fw[u][a] = *(const i8_v4*)(w[a] + k);
#pragma unroll
            for (int b = 0; b < MT; ++b) fx[u][b] = *(const i8_v4*)(x[b] + k);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (r + u < end) {
#pragma unroll
                for (int a = 0; a < NT; ++a)
#pragma unroll
                    for (int b = 0; b < MT; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u][a], fx[u][b], acc[a][b], 0, 0, 0);
            }
    }
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) s_part[wave][a * MT + b][lane] = acc[a][b];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * MT * NT; e += 64 * kWaves) {
        const int n = n0 + e % (16 * NT), m = e / (16 * NT);       // neighbouring threads: neighbouring channels of one token
        if (m >= A.rows || n >= A.cols) continue;
        const int nl = (n - n0) & 15, tile = ((n - n0) >> 4) * MT + (m >> 4), from = (nl >> 2) * 16 + (m & 15);
        int sum = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) sum += s_part[v][tile][from][nl & 3];
        ((T*)A.y)[(int64_t)m * A.ldy + n] = i8_finish<K>(i8_scaled<true>(sum, A.sx[m], A.sw[n]), A.bias ? A.bias[n] : 0.0f, A.bias != nullptr, A.relu != 0);
    }
}

// The same for very few rows of floats, rounded by every workgroup for itself into LDS, so that there is one launch and nothing to wait for:
// W's first operands are on their way meanwhile. Rows are dealt to groups of wavefronts; x is read twice, the second time from the
// cache. See i8_is_one for when.
template <int X, int K, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void k_linear_i8_one(const I8Args A, const I8Short B, int per_row)
{
    typedef typename I8Type<K>::T T;
    typedef typename I8Type<X>::T XT;
    constexpr int n = I8Piece<X>::n, kAhead = 8;
    __shared__ i8_v4 s_part[kWaves][64];
    __shared__ uint32_t s_top[kWaves];
    __shared__ float s_scale[kWaves];
    extern __shared__ __align__(16) int8_t s_x[];       // rows of inner + 16 codes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = lane & 15, q = lane >> 4;
    const int n0 = (int)blockIdx.x * 16;
    const int runs = A.inner >> 6, each = (runs + kWaves - 1) / kWaves, begin = wave * each, end = min(begin + each, runs);
    const int8_t* const w = A.w + (int64_t)blockIdx.x * runs * 1024 + lane * 16;
    i8_v4 fw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fw[u] = *(const i8_v4*)(w + (int64_t)max(min(begin + u, end - 1), 0) * 1024);

    const int row = wave / per_row, part = wave % per_row, stride = A.inner + 16;
    const bool mine = row < A.rows;
    const XT* const from = (const XT*)B.x + (int64_t)(mine ? row : 0) * B.ldx;
    auto get = [&](int k0, I8Piece<X>& v) {
        if (k0 + n <= B.inner) i8_get<X>(v, from + k0);
        else {
#pragma unroll
            for (int k = 0; k < n; ++k) v.v[k] = k0 + k < B.inner ? from[k0 + k] : I8Type<X>::down(0.0f);
        }
    };
    uint32_t top = 0;
    if (mine)
        for (int k0 = (part * 64 + lane) * n; k0 < B.inner; k0 += per_row * 64 * n) {
            I8Piece<X> v;
            get(k0, v);
#pragma unroll
            for (int k = 0; k < n; ++k) top = max(top, i8_bits(I8Type<X>::up(v.v[k])));
        }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    for (int p = 0; p < per_row; ++p) top = max(top, s_top[row * per_row + p]);
    float sc;
    const float factor = i8_factor(top, sc);
    const bool finite = top < 0x7f800000u;
    if (part == 0 && lane == 0) s_scale[row] = sc;
    if (mine)
        for (int k0 = (part * 64 + lane) * n; k0 < A.inner; k0 += per_row * 64 * n) {
            I8Piece<X> v;
            get(k0, v);
            uint32_t word[n / 4];
#pragma unroll
            for (int i = 0; i < n / 4; ++i) {
                word[i] = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) word[i] |= i8_code(I8Type<X>::up(v.v[4 * i + k]), factor, finite) << (8 * k);
            }
#pragma unroll
            for (int i = 0; i < n / 4; ++i) *(uint32_t*)(s_x + row * stride + k0 + 4 * i) = word[i];
        }
    __syncthreads();
    const int8_t* const x = s_x + min(t, A.rows - 1) * stride + q * 16;
    i8_v4 acc = {0, 0, 0, 0};
    for (int r = begin; r < end; r += kAhead) {
        if (r > begin) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) fw[u] = *(const i8_v4*)(w + (int64_t)min(r + u, end - 1) * 1024);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (r + u < end) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], *(const i8_v4*)(x + (r + u) * 64), acc, 0, 0, 0);
    }
    s_part[wave][lane] = acc;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int nl = threadIdx.x & 15, m = threadIdx.x >> 4;
    if (m >= A.rows || n0 + nl >= A.cols) return;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) sum += s_part[v][(nl >> 2) * 16 + m][nl & 3];
    ((T*)A.y)[(int64_t)m * A.ldy + n0 + nl] = i8_finish<K>(i8_scaled<true>(sum, s_scale[m], A.sw[n0 + nl]), A.bias ? A.bias[n0 + nl] : 0.0f, A.bias != nullptr, A.relu != 0);
}

static int i8_padded(int64_t cols) { return (int)(cols <= 64 ? 64 : (cols + 127) / 128 * 128); }

// ldq: row stride of the codes, or their padded length when they are packed
template <int K, bool kPacked>
static void i8_quantize(const void* xv, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, hipStream_t stream)
{
    typedef typename I8Type<K>::T T;
    const T* x = (const T*)xv;
    constexpr int n = I8Piece<K>::n;
    const bool pieces = (((uintptr_t)q | (uintptr_t)ldq) & 7u) == 0;
#define I8_ROWS(G, P)                                                                                                                  \
    hipLaunchKernelGGL((k_quantize_rows<K, kPacked, G, P>), i8_grid((rows + 256 / G - 1) / (256 / G)), dim3(256), 0, stream, x, rows, \
                       (int)cols, ldx, q, ldq, scale)
    if (!pieces || ldq > 256 * 8 * n)
        hipLaunchKernelGGL((k_quantize_rows_long<K, kPacked>), i8_grid(rows), dim3(256), 0, stream, x, rows, (int)cols, ldx, q, (int)ldq, scale);
    else if (ldq <= 16 * n) I8_ROWS(16, 1);
    else if (ldq <= 64 * n) I8_ROWS(64, 1);
    else if (ldq <= 64 * 4 * n) I8_ROWS(64, 4);
    else if (ldq <= 256 * 2 * n) I8_ROWS(256, 2);
    else if (ldq <= 256 * 4 * n) I8_ROWS(256, 4);
    else I8_ROWS(256, 8);
#undef I8_ROWS
}

template <bool kPacked>
static void i8_rows(const void* x, int x_type, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, hipStream_t stream)
{
    if (x_type == I8_F32) i8_quantize<I8_F32, kPacked>(x, rows, cols, ldx, q, ldq, scale, stream);
    else if (x_type == I8_F16) i8_quantize<I8_F16, kPacked>(x, rows, cols, ldx, q, ldq, scale, stream);
    else i8_quantize<I8_BF16, kPacked>(x, rows, cols, ldx, q, ldq, scale, stream);
}

static void i8_pack(const int8_t* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* packed, hipStream_t stream)
{
    const int64_t padded = i8_padded(cols), pieces = (rows + 15) / 16 * padded;
    hipLaunchKernelGGL(k_pack_rows, i8_grid((pieces + 255) / 256), dim3(256), 0, stream, x, rows, (int)cols, ldx, packed, padded, pieces);
}

// Rows of up to 256 values, where rounding them first (a launch, codes written and read again) costs more than reading x once for every 64
// channels. Captured calls, this way against the other: 100000 x 64 x 128 15 us against 50, 100000 x 128 x 256 40 against 72, 100000 x 256 x 256
// 81 against 63; 4000 x 128 x 128 4.4 against 6.0, 2000 x 512 x 128 4.7 against 6.1. Rows of up to 64 have no other way.
static bool i8_is_short(int64_t rows, int64_t cols, int64_t padded)
{
    return padded == 64 || (padded <= 256 && rows > 64 && (cols <= 192 || (cols <= 512 && rows <= 4096)));
}

// Workgroups of 256 threads of a kernel that the card holds at a time. The short rows' wavefronts walk over as many blocks each, so that
// no round is left half empty: 300000 x 64 x 32 16.6 us against 18.3 with 2048 workgroups, 100000 x 128 x 128 18.4 against 22.0,
// 100000 x 128 x 256 39.9 against 47.5.
template <typename F>
static int i8_resident(F kernel)
{
    int each = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, 256, 0) != hipSuccess || each < 1) each = 4;
    return 256 * each;
}

template <int X, int K, int KS>
static void i8_short_of(const I8Args& A, const I8Short& B, hipStream_t stream)
{
    static const int resident = i8_resident(k_linear_i8_short<X, K, KS>);
    const dim3 grid((unsigned)std::min<int64_t>(((int64_t)A.rows + 63) / 64, resident), (unsigned)((A.cols + 63) / 64));
    hipLaunchKernelGGL((k_linear_i8_short<X, K, KS>), grid, dim3(256), 0, stream, A, B);
}

template <int X, int K>
static void i8_short(const I8Args& A, const I8Short& B, hipStream_t stream)
{
    if (A.inner == 64) i8_short_of<X, K, 1>(A, B, stream);
    else if (A.inner == 128) i8_short_of<X, K, 2>(A, B, stream);
    else i8_short_of<X, K, 4>(A, B, stream);
}

// Very few rows, by the time of the captured call against rounding in a launch before: 1 x 4096 x 4096 6.6 us against 8.4, 1 x 4096 x 14336
// 16.5 against 19.4, 2 x 4096 x 4096 7.5 against 8.4, 8 x 1024 x 1024 4.5 against 5.6; but 4 x 4096 x 4096 8.8 against 8.3 and
// 4 x 28672 x 4096 36 against 27, each workgroup's share of the rounding growing with the rows.
static bool i8_is_one(int64_t rows, int64_t padded, int x_type)
{
    return x_type != I8_INT8 && rows <= 8 && rows * padded <= (rows == 1 ? 32768 : 8192);
}

template <int X, int K>
static void i8_one(const I8Args& A, const I8Short& B, hipStream_t stream)
{
    const dim3 grid((unsigned)((A.cols + 15) / 16));
    const int groups = A.rows <= 1 ? 1 : A.rows <= 2 ? 2 : A.rows <= 4 ? 4 : 8;
    hipLaunchKernelGGL((k_linear_i8_one<X, K, 8>), grid, dim3(512), (size_t)A.rows * (A.inner + 16), stream, A, B, 8 / groups);
}

template <int K, int MT, int NT>
static void i8_few(const I8Args& A, hipStream_t stream)
{
    const dim3 grid((unsigned)((A.cols + 16 * NT - 1) / (16 * NT)));
    if (A.inner >= 2048) hipLaunchKernelGGL((k_linear_i8_few<K, MT, NT, 8>), grid, dim3(512), 0, stream, A);
    else hipLaunchKernelGGL((k_linear_i8_few<K, MT, NT, 4>), grid, dim3(256), 0, stream, A);
}

template <int K, int TM, int TN, int WN, int R>
static int i8_tiles(const I8Args& A, hipStream_t stream)
{
    const int64_t tiles = (int64_t)((A.rows + 64 * TM - 1) / (64 * TM)) * ((A.cols + 32 * TN * WN - 1) / (32 * TN * WN));
    if (tiles * 128 * WN >= (int64_t)1 << 32) {
        hrf_set_error("hrf_linear_int8: too many tiles");
        return 1;
    }
    hipLaunchKernelGGL((k_linear_i8<K, TM, TN, WN, R>), dim3((unsigned)tiles), dim3(128 * WN), 0, stream, A);
    return 0;
}

#define I8_FEW 64       // rows up to which the product of few tokens runs, on packed codes

template <int K>
static int i8_linear(const I8Args& A, hipStream_t stream)
{
    if (A.rows <= 16) { i8_few<K, 1, 1>(A, stream); return 0; }
    if (A.rows <= 32) { i8_few<K, 2, 2>(A, stream); return 0; }
    if (A.rows <= I8_FEW) { i8_few<K, 4, 2>(A, stream); return 0; }
    // Rounds of the card times what a round of that size takes against one of 128 x 128: larger tiles read each operand less often, smaller ones
    // fill the card when there is little, and a round that only a few tiles need takes as long as a full one (264 tiles of 128 on 256
    // CUs: two). Captured calls in us, rounding included, with 64 / 128 / 128 x 192 / 256:
    //   219 x 71 x 5967   17 / 28 / 31 / 60      1237 x 2827 x 5225  50 / 35 / 39 / 63      1021 x 4099 x 2051  29 / 30 / 25 / 40
    //   325 x 4341 x 6165 35 / 40 / 47 / 68      11905 x 625 x 1683  46 / 38 / 43 / 43      1000 x 5000 x 3000  39 / 34 / 30 / 43
    //   4096^3           125 / 92 / 87 / 74      8192^3            1032 / 674 / 677 / 512   8192 x 8192 x 512  121 / 80 / 91 / 77
    // (64 x 64 with 128 bytes of k a stage: with 64 bytes the first takes 24.) Below 512 k the ends count, which a CU overlaps for two
    // of the smaller tiles: 6465 x 1799 x 214 27 / 21 / 24 / 23.
    auto rounds = [&](int m, int n) { return (((int64_t)A.rows + m - 1) / m * (((int64_t)A.cols + n - 1) / n) + 255) / 256; };
    const int64_t c64 = 9 * rounds(64, 64), c128 = 20 * rounds(128, 128), c192 = 25 * rounds(128, 192), c256 = 60 * rounds(256, 256);
    if (A.inner >= 512 && c256 < std::min(std::min(c64, c128), c192)) return i8_tiles<K, 4, 2, 4, 1>(A, stream);
    if (A.inner >= 512 && c192 < std::min(c64, c128)) return i8_tiles<K, 2, 3, 2, 1>(A, stream);
    if (c128 < c64) return i8_tiles<K, 2, 2, 2, 1>(A, stream);
    return i8_tiles<K, 1, 1, 2, 2>(A, stream);
}

template <int K>
static int i8_product(I8Args& A, const void* x, int x_type, int64_t ldx, const float* x_scale, int inner, void* workspace, hipStream_t stream)
{
    if (i8_is_short(A.rows, A.cols, A.inner)) {
        I8Short B;
        B.x = x; B.ldx = ldx; B.sx = x_scale; B.inner = inner;
        if (x_type == I8_F32) i8_short<I8_F32, K>(A, B, stream);
        else if (x_type == I8_F16) i8_short<I8_F16, K>(A, B, stream);
        else if (x_type == I8_BF16) i8_short<I8_BF16, K>(A, B, stream);
        else i8_short<I8_INT8, K>(A, B, stream);
        return 0;
    }
    if (i8_is_one(A.rows, A.inner, x_type)) {
        I8Short B;
        B.x = x; B.ldx = ldx; B.sx = nullptr; B.inner = inner;
        if (x_type == I8_F32) i8_one<I8_F32, K>(A, B, stream);
        else if (x_type == I8_F16) i8_one<I8_F16, K>(A, B, stream);
        else i8_one<I8_BF16, K>(A, B, stream);
        return 0;
    }
    float* const scale = (float*)((int8_t*)workspace + ((int64_t)A.rows + 15) / 16 * 16 * A.inner);
    A.x = (const int8_t*)workspace;
    A.ldx = A.inner;
    A.sx = x_type == I8_INT8 ? x_scale : scale;
    const bool few = A.rows <= I8_FEW;
    if (x_type != I8_INT8) {
        if (few) i8_rows<true>(x, x_type, A.rows, inner, ldx, (int8_t*)workspace, A.inner, scale, stream);
        else i8_rows<false>(x, x_type, A.rows, inner, ldx, (int8_t*)workspace, A.inner, scale, stream);
    } else if (few) {
        i8_pack((const int8_t*)x, A.rows, inner, ldx, (int8_t*)workspace, stream);
    } else if (inner == A.inner && (((uintptr_t)x | (uintptr_t)ldx) & 15u) == 0 && ldx < (1 << 23)) {
        A.x = (const int8_t*)x;         // rows that lie as the tiles read them
        A.ldx = ldx;
    } else {
        hipLaunchKernelGGL(k_pad_rows, i8_grid(A.rows), dim3(256), 0, stream, (const int8_t*)x, (int64_t)A.rows, inner, ldx, (int8_t*)workspace, A.inner);
    }
    const hipError_t rounded = hipGetLastError();       // (no product of codes that nobody wrote)
    if (rounded != hipSuccess) {
        hrf_set_error("hrf_linear_int8: launch failed: %s", hipGetErrorString(rounded));
        return 2;
    }
    return i8_linear<K>(A, stream);
}

static bool i8_inner_ok(int64_t inner) { return inner >= 1 && inner <= HRF_INT8_MAX_INNER; }

extern "C" int64_t hrf_int8_padded(int64_t inner) { return i8_inner_ok(inner) ? i8_padded(inner) : -1; }

extern "C" int64_t hrf_int8_packed_bytes(int64_t rows, int64_t inner) { return rows < 0 || !i8_inner_ok(inner) ? -1 : (rows + 15) / 16 * 16 * i8_padded(inner); }

extern "C" int64_t hrf_linear_int8_workspace_bytes(int64_t rows, int64_t cols, int64_t inner)
{
    if (rows <= 0 || cols <= 0 || !i8_inner_ok(inner) || i8_is_short(rows, cols, i8_padded(inner))) return 0;
    return hrf_int8_packed_bytes(rows, inner) + rows * 4;
}

extern "C" int hrf_quantize_rows_int8(const void* x, int x_type, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                                      float* scale, hrf_stream_t stream)
{
    HRF_CHECK_ARG(x_type >= I8_F32 && x_type <= I8_BF16, "x_type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    HRF_CHECK_ARG(rows >= 0 && rows < HRF_INT8_MAX_ROWS && i8_inner_ok(cols), "bad sizes");
    if (rows == 0) return 0;
    HRF_CHECK_ARG(x && q && scale, "NULL argument");
    HRF_CHECK_ARG((ldx >= cols || rows == 1) && ldq >= cols && ldq <= HRF_INT8_MAX_INNER + 1, "a row stride is shorter than the row, or that of q too long");
    i8_rows<false>(x, x_type, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}

extern "C" int hrf_int8_pack(const int8_t* q, int64_t rows, int64_t cols, int64_t ldq, int8_t* packed, hrf_stream_t stream)
{
    HRF_CHECK_ARG(rows >= 0 && rows < HRF_INT8_MAX_ROWS && i8_inner_ok(cols), "bad sizes");
    if (rows == 0) return 0;
    HRF_CHECK_ARG(q && packed, "NULL argument");
    HRF_CHECK_ARG(ldq >= cols || rows == 1, "a row stride is shorter than the row");
    HRF_CHECK_ARG(((uintptr_t)packed & 15u) == 0, "the packed codes must begin at a multiple of 16 bytes");
    i8_pack(q, rows, cols, ldq, packed, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}

extern "C" int hrf_linear_int8(const void* x, int x_type, int64_t ldx, const float* x_scale, const int8_t* w, const float* w_scale,
                               const float* bias, int64_t rows, int64_t cols, int64_t inner, void* y, int y_type, int64_t ldy, int relu,
                               void* workspace, hrf_stream_t stream)
{
    HRF_CHECK_ARG(x_type >= I8_F32 && x_type <= I8_INT8, "x_type must be 0 (fp32), 1 (fp16), 2 (bf16) or 3 (int8)");
    HRF_CHECK_ARG(y_type >= I8_F32 && y_type <= I8_BF16, "y_type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    HRF_CHECK_ARG(rows >= 0 && rows < HRF_INT8_MAX_ROWS && cols >= 0 && cols <= 64 * 65535 && i8_inner_ok(inner), "bad sizes");
    HRF_CHECK_ARG(((rows + 127) / 128) * ((cols + 127) / 128) < ((int64_t)1 << 31) && hrf_int8_packed_bytes(rows, inner) < ((int64_t)1 << 42), "too many tiles");
    if (rows == 0 || cols == 0) return 0;
    HRF_CHECK_ARG(x && w && w_scale && y && (x_scale || x_type != I8_INT8), "NULL argument");
    HRF_CHECK_ARG((ldx >= inner || rows == 1) && (ldy >= cols || rows == 1), "a row stride is shorter than the row");
    HRF_CHECK_ARG(((uintptr_t)w & 15u) == 0, "w must begin at a multiple of 16 bytes");
    HRF_CHECK_ARG(hrf_linear_int8_workspace_bytes(rows, cols, inner) == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0),
                  "the workspace must begin at a multiple of 16 bytes");
    I8Args A;
    A.x = nullptr; A.ldx = 0; A.w = w; A.sx = nullptr; A.sw = w_scale; A.bias = bias; A.y = y; A.ldy = ldy;
    A.rows = (int)rows; A.cols = (int)cols; A.inner = i8_padded(inner); A.relu = relu;
    int rc;
    if (y_type == I8_F32) rc = i8_product<I8_F32>(A, x, x_type, ldx, x_scale, (int)inner, workspace, (hipStream_t)stream);
    else if (y_type == I8_F16) rc = i8_product<I8_F16>(A, x, x_type, ldx, x_scale, (int)inner, workspace, (hipStream_t)stream);
    else rc = i8_product<I8_BF16>(A, x, x_type, ldx, x_scale, (int)inner, workspace, (hipStream_t)stream);
    if (rc != 0) return rc;
    HRF_CHECK_LAUNCH();
    return 0;
}
