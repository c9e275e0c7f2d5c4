// Matrix product in 8-bit integers with a scale for each token (row of x) and each channel (row of W), and the rounding of rows to 8 bits.
//
//   y[m][n] = act( (sum_k xq[m][k] wq[n][k]) * sx[m] * sw[n] + bias[n] )        xq, wq in -128 .. 127, sums exact in int32
//   row -> codes: s = amax * (1 / 127), q = rint(x * (127 / amax)), amax = max(max |x|, 2^-119)
//
// The sums are v_mfma_i32_16x16x64_i8: 16 bytes a lane and operand, row (lane & 15), bytes 16 (lane >> 4) .. + 15 of 64. The order of k
// inside an instruction is the same for both operands, so it does not matter; the result's rows are W's channels, its columns x's tokens
// (lane & 15), and a lane's four values are four consecutive channels of one token.
// Rows of both operands begin at multiples of 16 bytes and are padded with zeros to a multiple of 64 (128 when longer than 64): a product
// with padding is the product. Epilogue in fp32, one rounding per operation, one to the type of y.
#include "hrf_common.h"
#include <algorithm>

enum { I8_F32 = 0, I8_F16 = 1, I8_BF16 = 2, I8_INT8 = 3 };

typedef int i8_v4 __attribute__((ext_vector_type(4)));
#define I8_GLOBAL __attribute__((address_space(1)))
#define I8_LDS __attribute__((address_space(3)))

template <int K> struct I8Type;
template <> struct I8Type<I8_F32> { typedef float T; static __device__ float up(float x) { return x; } static __device__ float down(float x) { return x; } };
template <> struct I8Type<I8_F16> { typedef __half T; static __device__ float up(__half x) { return __half2float(x); } static __device__ __half down(float x) { return __float2half_rn(x); } };
template <> struct I8Type<I8_BF16> { typedef __bf16 T; static __device__ float up(__bf16 x) { return (float)x; } static __device__ __bf16 down(float x) { return (__bf16)x; } };

// ------------------------------------------------------------------------------------------------ rows -> codes and scales
// One 16-byte piece of a row, as fp32.
template <int K> struct alignas(16) I8Piece { static constexpr int n = 16 / (int)sizeof(typename I8Type<K>::T); typename I8Type<K>::T v[16 / sizeof(typename I8Type<K>::T)]; };

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

// kGroup lanes (a power of two, or the whole workgroup of 256 in groups of 64 joined through LDS) a row; the row is read once and stays in
// registers, kPieces 16-byte pieces a lane. Both sides of that: rows of 4096 bf16 from memory twice, value by value, 118 us for 8192
// of them; this way 35 us.
template <int K, int kGroup, int kPieces>
__global__ __launch_bounds__(256) void k_quantize_rows(const typename I8Type<K>::T* __restrict__ x, int64_t rows, int cols, int64_t ldx,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale)
{
    __shared__ uint32_t s_max[4];
    constexpr int n = I8Piece<K>::n, kRows = 256 / kGroup;
    const int lane = threadIdx.x % kGroup;
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kGroup;
    const bool here = row < rows;
    const typename I8Type<K>::T* const from = x + (here ? row : rows - 1) * ldx;
    I8Piece<K> v[kPieces];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        const int k0 = (p * kGroup + lane) * n;
        if (k0 + n <= cols) v[p] = *(const I8Piece<K>*)(from + k0);
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
    int8_t* const to = q + row * ldq;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        const int k0 = (p * kGroup + lane) * n;
        if (k0 >= ldq) continue;        // (the padding up to ldq is a multiple of 64 away: whole pieces)
        uint32_t word[n / 4];
#pragma unroll
        for (int w = 0; w < n / 4; ++w) {
            word[w] = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) word[w] |= i8_code(I8Type<K>::up(v[p].v[4 * w + k]), factor, finite) << (8 * k);
        }
        if (n == 8) *(uint2*)(to + k0) = make_uint2(word[0], word[n / 4 - 1]);
        else *(uint32_t*)(to + k0) = word[0];
    }
}

// Rows at addresses that are no multiples of 16 bytes, or longer than 16384: value by value, twice.
template <int K>
__global__ __launch_bounds__(256) void k_quantize_rows_any(const typename I8Type<K>::T* __restrict__ x, int64_t cols, int64_t ldx,
                                                           int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale)
{
    __shared__ uint32_t s_max[4];
    x += (int64_t)blockIdx.x * ldx;
    q += (int64_t)blockIdx.x * ldq;
    uint32_t top = 0;
    for (int64_t k = threadIdx.x; k < cols; k += 256) top = max(top, i8_bits(I8Type<K>::up(x[k])));
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    float sc;
    const float factor = i8_factor(top, sc);
    const bool finite = top < 0x7f800000u;
    if (threadIdx.x == 0) scale[blockIdx.x] = sc;
    for (int64_t k = threadIdx.x; k < ldq; k += 256) q[k] = k < cols ? (int8_t)i8_code(I8Type<K>::up(x[k]), factor, finite) : (int8_t)0;
}

__global__ __launch_bounds__(256) void k_pad_rows(const int8_t* __restrict__ x, int64_t cols, int64_t ldx, int8_t* __restrict__ q, int64_t ldq)
{
    x += (int64_t)blockIdx.x * ldx;
    q += (int64_t)blockIdx.x * ldq;
    for (int64_t k = threadIdx.x; k < ldq; k += 256) q[k] = k < cols ? x[k] : (int8_t)0;
}

// ------------------------------------------------------------------------------------------------ product
struct I8Args {
    const int8_t* x;
    const int8_t* w;
    const float* sx;
    const float* sw;
    const float* bias;
    void* y;
    int64_t ldx, ldw, ldy;
    int rows, cols, inner;      // inner: padded
    int relu;
};

template <int K>
__device__ __forceinline__ typename I8Type<K>::T i8_finish(int acc, float sx, float sw, float bias, bool has_bias, bool relu)
{
    float v = (float)acc * (sx * sw);       // (a product of scales overflows only where the output does)
    if (has_bias) v = v + bias;
    if (relu) v = v < 0.0f ? 0.0f : v;
    return I8Type<K>::down(v);
}

// 16 bytes from base + offset (each lane its own) to LDS, the wavefront's kilobyte from byte `to` on in the order of its lanes. The
// compiler takes the builtin for this as something every later LDS read may depend on and waits for it at once; here the caller waits
// (s_waitcnt vmcnt, a barrier) before anybody reads. No register is written but m0, which the compiler never keeps a value in.
__device__ __forceinline__ void i8_load_lds(const int8_t* base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
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

// Tiles of BM = 64 TM tokens x BN = 64 TN channels, four wavefronts 2 x 2, 32 TM x 32 TN each from v_mfma_i32_32x32x32_i8. A stage is 128
// bytes of k in LDS, two stages, filled by direct loads (16 bytes a lane, no registers). A row's eight 16-byte chunks lie in LDS permuted
// by its number, so that lanes that read the same chunk of neighbouring rows hit all banks.
// The operands of the next 32 k are read from LDS while the matrix cores work on these; before the last 32 k of a stage the workgroup
// meets, the loads of the stage after the next take the buffer that everybody has read, and the next stage's first operands follow.
template <int K, int TM, int TN>
__global__ __launch_bounds__(256, (TM * TN > 8 ? 1 : 2)) void k_linear_i8(const I8Args A)
{
    constexpr int BM = 64 * TM, BN = 64 * TN, kStage = (BM + BN) * 128, kLoads = (BM + BN) / 32;
    typedef typename I8Type<K>::T T;
    typedef int i8_v16 __attribute__((ext_vector_type(16)));
    __shared__ __align__(16) int8_t s_tile[2 * kStage];
    __shared__ float s_sx[BM], s_sw[BN], s_bias[BN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    int tm, tn;
    i8_tile_of((A.rows + BM - 1) / BM, (A.cols + BN - 1) / BN, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int8_t* const xb = A.x + (int64_t)m0 * A.ldx;
    const int8_t* const wb = A.w + (int64_t)n0 * A.ldw;
    const int steps = A.inner >> 7;

    // this lane's part of each load: row first + lane / 8 of the stage (rows past the end read the last one), its chunk permuted
    uint32_t from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int first = (wave * kLoads + i) * 8, r = first + (lane >> 3), chunk = (lane & 7) ^ ((lane >> 3) & 7);
        from[i] = (first < BM ? (uint32_t)min(r, A.rows - 1 - m0) * (uint32_t)A.ldx : (uint32_t)min(r - BM, A.cols - 1 - n0) * (uint32_t)A.ldw) + chunk * 16;
    }
    const uint32_t lds = (uint32_t)(uintptr_t)(I8_LDS int8_t*)s_tile;
    auto load = [&](int i, int buf, int k0) {
        const int first = (wave * kLoads + i) * 8;
        i8_load_lds((first < BM ? xb : wb) + k0, from[i], lds + buf * kStage + first * 128);
    };
    i8_v16 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[a][b][k] = 0;
    i8_v4 fx[2][TM], fw[2][TN];
    const int x_row = (wm * 32 * TM + (lane & 31)) * 128, w_row = (BM + wn * 32 * TN + (lane & 31)) * 128;
    auto read = [&](int set, int buf, int kk) {
        const int chunk = ((kk * 2 + (lane >> 5)) ^ (lane & 7)) * 16;
        const int8_t* t = s_tile + buf * kStage + chunk;
#pragma unroll
        for (int b = 0; b < TM; ++b) fx[set][b] = *(const i8_v4*)(t + x_row + b * 32 * 128);
#pragma unroll
        for (int a = 0; a < TN; ++a) fw[set][a] = *(const i8_v4*)(t + w_row + a * 32 * 128);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][a], fx[set][b], acc[a][b], 0, 0, 0);
    };
    for (int k = threadIdx.x; k < BM; k += 256) s_sx[k] = A.sx[min(m0 + k, A.rows - 1)];
    for (int k = threadIdx.x; k < BN; k += 256) {
        const int n = min(n0 + k, A.cols - 1);
        s_sw[k] = A.sw[n];
        s_bias[k] = A.bias ? A.bias[n] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(i, 0, 0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 1) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(i, 1, 128);
    }
    read(0, 0, 0);
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
#pragma unroll
        for (int kk = 0; kk < 3; ++kk) {
            read((kk + 1) & 1, buf, kk + 1);
            multiply(kk & 1);
#ifndef NO_SGB
#pragma unroll
            for (int i = 0; i < TM + TN; ++i) {     // one operand read for every TM TN / (TM + TN) products
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, TM * TN / (TM + TN), 0);
            }
#endif
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");     // the next stage has landed, this one is in registers
        if (s + 1 < steps) read(0, buf ^ 1, 0);
        if (s + 2 < steps) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(i, buf, (s + 2) << 7);
        }
        multiply(1);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // Epilogue: through LDS, so that a row of y leaves in 16-byte pieces side by side. Pieces lie permuted by their row's number again.
    constexpr int kPer = 16 / (int)sizeof(T), kPieces = BN / kPer;          // values a piece, pieces a row
    constexpr int kPasses = BM * BN * (int)sizeof(T) > 2 * kStage ? 2 : 1, kRows = BM / kPasses;
    T* const out = (T*)s_tile;
    const bool has_bias = A.bias != nullptr, relu = A.relu != 0;
    const bool wide = (((uintptr_t)A.y | (uintptr_t)(A.ldy * (int64_t)sizeof(T))) & 15u) == 0;
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        if (kPasses == 1 || wm == pass) {
#pragma unroll
            for (int b = 0; b < TM; ++b) {
                const int ml = wm * 32 * TM + b * 32 + (lane & 31), row = ml - pass * kRows;
                const float sx = s_sx[ml];
#pragma unroll
                for (int a = 0; a < TN; ++a)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int nl = wn * 32 * TN + a * 32 + g * 8 + (lane >> 5) * 4;
                        T v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = i8_finish<K>(acc[a][b][g * 4 + k], sx, s_sw[nl + k], s_bias[nl + k], has_bias, relu);
                        T* to = out + row * BN + ((nl / kPer) ^ (row & (kPieces - 1))) * kPer + nl % kPer;
                        if (sizeof(T) == 4) *(i8_v4*)to = *(const i8_v4*)v;
                        else *(uint64_t*)to = *(const uint64_t*)v;
                    }
            }
        }
        __syncthreads();
        for (int p = threadIdx.x; p < kRows * kPieces; p += 256) {
            const int row = p / kPieces, piece = p % kPieces;
            const int m = m0 + pass * kRows + row, n = n0 + piece * kPer;
            if (m >= A.rows || n >= A.cols) continue;
            const T* v = out + row * BN + (piece ^ (row & (kPieces - 1))) * kPer;
            T* y = (T*)A.y + (int64_t)m * A.ldy + n;
            if (wide && n + kPer <= A.cols) *(i8_v4*)y = *(const i8_v4*)v;
            else
                for (int k = 0; k < kPer && n + k < A.cols; ++k) y[k] = v[k];
        }
        if (pass + 1 < kPasses) __syncthreads();
    }
}

// Short rows (up to 64 KS values), many of them: bound by the bytes of x and y, so x is rounded on its way in and nothing is written
// between. A wavefront keeps the weights of 64 channels in registers and walks over blocks of 16 tokens; lane (t, q) = (lane & 15, lane >> 4)
// holds 16 values of token t for each 64, finds the row's largest with the three other lanes of the token, and has its operand. The
// channels are dealt to the instructions so that a lane's 16 results are 16 neighbouring channels of one token: 32 bytes of fp16 in a
// row of 128.
struct I8Short {
    const void* x;
    int64_t ldx;
    int inner;              // not padded
    int x_wide, y_wide;     // rows of x / y begin at multiples of 16 bytes
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
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int row = min(n0 + (t >> 2) * 16 + a * 4 + (t & 3), A.cols - 1);
#pragma unroll
        for (int s = 0; s < KS; ++s) fw[s][a] = *(const i8_v4*)(A.w + (int64_t)row * A.ldw + s * 64 + q * 16);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int n = min(n0 + q * 16 + k, A.cols - 1);
        sw[k] = A.sw[n];
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
            for (int s = 0; s < KS; ++s) fx[s] = *(const i8_v4*)((const int8_t*)B.x + row * B.ldx + s * 64 + q * 16);
            sx = A.sx[row];
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
                    if (B.x_wide && k0 + n <= B.inner) v[s][p] = *(const I8Piece<X>*)(from + k0);
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
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            i8_v4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[s][a], fx[s], acc, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[a * 4 + k] = i8_finish<K>(acc[k], sx, sw[a * 4 + k], bias[a * 4 + k], has_bias, relu);
        }
        if (m >= A.rows) continue;
        const int n = n0 + q * 16;
        T* const y = (T*)A.y + row * A.ldy + n;
        if (B.y_wide && n + 16 <= A.cols) {
#pragma unroll
            for (int p = 0; p < (int)sizeof(T); ++p) ((i8_v4*)y)[p] = ((const i8_v4*)out)[p];
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (n + k < A.cols) y[k] = out[k];
        }
    }
}

// Few tokens (up to 16 MT): bound by the bytes of W, which every workgroup reads its part of once: 16 NT channels, the k axis dealt to its
// kWaves wavefronts in runs of 64 bytes, sums joined in LDS. Integer sums: any order gives the same.
template <int K, int MT, int NT, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void k_linear_i8_few(const I8Args A)
{
    typedef typename I8Type<K>::T T;
    __shared__ i8_v4 s_part[kWaves][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = lane & 15, q = lane >> 4;
    const int n0 = (int)blockIdx.x * 16 * NT;
    const int runs = A.inner >> 6, each = (runs + kWaves - 1) / kWaves, begin = wave * each, end = min(begin + each, runs);
    const int8_t* w[NT];
    const int8_t* x[MT];
#pragma unroll
    for (int a = 0; a < NT; ++a) w[a] = A.w + (int64_t)min(n0 + a * 16 + t, A.cols - 1) * A.ldw + q * 16;
#pragma unroll
    for (int b = 0; b < MT; ++b) x[b] = A.x + (int64_t)min(b * 16 + t, A.rows - 1) * A.ldx + q * 16;
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
            const int64_t k = (int64_t)min(r + u, end - 1) * 64;
#pragma unroll
            for (int a = 0; a < NT; ++a) fw[u][a] = __builtin_nontemporal_load((const i8_v4*)(w[a] + k));
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
        ((T*)A.y)[(int64_t)m * A.ldy + n] = i8_finish<K>(sum, A.sx[m], A.sw[n], A.bias ? A.bias[n] : 0.0f, A.bias != nullptr, A.relu != 0);
    }
}

template <int K>
static void i8_quantize(const void* xv, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, hipStream_t stream)
{
    typedef typename I8Type<K>::T T;
    const T* x = (const T*)xv;
    constexpr int n = I8Piece<K>::n;
    const int64_t width = std::max(cols, ldq);
    // whole pieces: rows of x at multiples of 16 bytes, rows of q at multiples of 8 and padded to them
    const bool pieces = (((uintptr_t)x | (uintptr_t)(ldx * (int64_t)sizeof(T))) & 15u) == 0 && (((uintptr_t)q | (uintptr_t)ldq) & 7u) == 0;
#define I8_ROWS(G, P)                                                                                                            \
    hipLaunchKernelGGL((k_quantize_rows<K, G, P>), dim3((unsigned)((rows + 256 / G - 1) / (256 / G))), dim3(256), 0, stream, x, rows, \
                       (int)cols, ldx, q, ldq, scale)
    if (!pieces || width > 256 * 8 * n)
        hipLaunchKernelGGL(k_quantize_rows_any<K>, dim3((unsigned)rows), dim3(256), 0, stream, x, cols, ldx, q, ldq, scale);
    else if (width <= 16 * n) I8_ROWS(16, 1);
    else if (width <= 64 * n) I8_ROWS(64, 1);
    else if (width <= 64 * 4 * n) I8_ROWS(64, 4);
    else if (width <= 256 * 4 * n) I8_ROWS(256, 4);
    else I8_ROWS(256, 8);
#undef I8_ROWS
}

static int i8_padded(int64_t cols) { return (int)(cols <= 64 ? 64 : (cols + 127) / 128 * 128); }

extern "C" int64_t hrf_int8_padded(int64_t cols) { return cols < 1 || cols > HRF_INT8_MAX_INNER ? -1 : i8_padded(cols); }

extern "C" int hrf_quantize_rows_int8(const void* x, int x_type, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                                      float* scale, hrf_stream_t stream)
{
    HRF_CHECK_ARG(x_type >= I8_F32 && x_type <= I8_INT8, "x_type must be 0 (fp32), 1 (fp16), 2 (bf16) or 3 (int8)");
    HRF_CHECK_ARG(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= HRF_INT8_MAX_INNER, "bad sizes");
    if (rows == 0) return 0;
    HRF_CHECK_ARG(x && q && (scale || x_type == I8_INT8), "NULL argument");
    HRF_CHECK_ARG((ldx >= cols || rows == 1) && ldq >= cols, "a row stride is shorter than the row");
    if (x_type == I8_F32) i8_quantize<I8_F32>(x, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream);
    else if (x_type == I8_F16) i8_quantize<I8_F16>(x, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream);
    else if (x_type == I8_BF16) i8_quantize<I8_BF16>(x, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream);
    else hipLaunchKernelGGL(k_pad_rows, dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream, (const int8_t*)x, cols, ldx, q, ldq);
    HRF_CHECK_LAUNCH();
    return 0;
}

static bool i8_wide(const void* p, int64_t ld, int size) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & 15u) == 0; }

// Rows of up to 256 values and up to 128 channels, when there are enough rows to fill the card.
static bool i8_is_short(int64_t rows, int64_t cols, int64_t inner) { return inner == 64 || (inner <= 256 && cols <= 128 && rows > 4096); }

template <int X, int K>
static void i8_short(const I8Args& A, const void* x, int64_t ldx, int64_t inner, int size, hipStream_t stream)
{
    I8Short B;
    B.x = x; B.ldx = ldx; B.inner = (int)inner; B.x_wide = i8_wide(x, ldx, size); B.y_wide = i8_wide(A.y, A.ldy, (int)sizeof(typename I8Type<K>::T));
    const dim3 grid((unsigned)std::min<int64_t>((A.rows + 63) / 64, 2048), (unsigned)((A.cols + 63) / 64));
    if (A.inner == 64) hipLaunchKernelGGL((k_linear_i8_short<X, K, 1>), grid, dim3(256), 0, stream, A, B);
    else if (A.inner == 128) hipLaunchKernelGGL((k_linear_i8_short<X, K, 2>), grid, dim3(256), 0, stream, A, B);
    else hipLaunchKernelGGL((k_linear_i8_short<X, K, 4>), grid, dim3(256), 0, stream, A, B);
}

template <int K, int MT, int NT>
static void i8_few(const I8Args& A, hipStream_t stream)
{
    const dim3 grid((unsigned)((A.cols + 16 * NT - 1) / (16 * NT)));
    if (A.inner >= 2048) hipLaunchKernelGGL((k_linear_i8_few<K, MT, NT, 8>), grid, dim3(512), 0, stream, A);
    else hipLaunchKernelGGL((k_linear_i8_few<K, MT, NT, 4>), grid, dim3(256), 0, stream, A);
}

template <int K>
static void i8_linear(const I8Args& A, hipStream_t stream)
{
    if (i8_is_short(A.rows, A.cols, A.inner)) { i8_short<I8_INT8, K>(A, A.x, A.ldx, A.inner, 1, stream); return; }
    if (A.rows <= 16) { i8_few<K, 1, 1>(A, stream); return; }
    if (A.rows <= 32) { i8_few<K, 2, 2>(A, stream); return; }
    if (A.rows <= 64) { i8_few<K, 4, 2>(A, stream); return; }
    const int64_t large = (int64_t)((A.rows + 255) / 256) * ((A.cols + 255) / 256);
    if (large >= 200) hipLaunchKernelGGL((k_linear_i8<K, 4, 4>), dim3((unsigned)large), dim3(256), 0, stream, A);
    else {
        const int64_t tiles = (int64_t)((A.rows + 127) / 128) * ((A.cols + 127) / 128);
        hipLaunchKernelGGL((k_linear_i8<K, 2, 2>), dim3((unsigned)tiles), dim3(256), 0, stream, A);
    }
}

#define I8_CHECK(cond, msg)                      \
    do {                                         \
        if (!(cond)) {                           \
            hrf_set_error("%s: %s", name, msg);  \
            return 1;                            \
        }                                        \
    } while (0)
static int i8_check(const char* name, const void* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                    int64_t rows, int64_t cols, int64_t inner, const void* y, int y_type, int64_t ldy)
{
    I8_CHECK(y_type >= I8_F32 && y_type <= I8_BF16, "y_type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    I8_CHECK(rows >= 0 && rows < ((int64_t)1 << 31) - 256 && cols >= 0 && cols < ((int64_t)1 << 31) - 256, "bad sizes");
    I8_CHECK(inner >= 64 && inner <= HRF_INT8_MAX_INNER + 1 && inner == i8_padded(inner), "inner must be a padded length (hrf_int8_padded)");
    if (rows == 0 || cols == 0) return 0;
    I8_CHECK(x && x_scale && w && w_scale && y, "NULL argument");
    I8_CHECK((ldx >= inner || rows == 1) && (ldw >= inner || cols == 1) && (ldy >= cols || rows == 1), "a row stride is shorter than the row");
    I8_CHECK((((uintptr_t)x | (uintptr_t)w) & 15u) == 0 && ((ldx | ldw) & 15) == 0, "x and w and their rows must begin at multiples of 16 bytes");
    I8_CHECK(ldx < HRF_INT8_MAX_STRIDE && ldw < HRF_INT8_MAX_STRIDE, "rows are too far apart");
    I8_CHECK(((rows + 127) / 128) * ((cols + 127) / 128) < ((int64_t)1 << 31) && cols <= 64 * 65535, "too many tiles");
    return 0;
}

extern "C" int hrf_linear_int8(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                               const float* bias, int64_t rows, int64_t cols, int64_t inner, void* y, int y_type, int64_t ldy, int relu,
                               hrf_stream_t stream)
{
    const int rc = i8_check(__func__, x, ldx, x_scale, w, ldw, w_scale, rows, cols, inner, y, y_type, ldy);
    if (rc || rows == 0 || cols == 0) return rc;
    I8Args A;
    A.x = x; A.w = w; A.sx = x_scale; A.sw = w_scale; A.bias = bias; A.y = y; A.ldx = ldx; A.ldw = ldw; A.ldy = ldy;
    A.rows = (int)rows; A.cols = (int)cols; A.inner = (int)inner; A.relu = relu;
    if (y_type == I8_F32) i8_linear<I8_F32>(A, (hipStream_t)stream);
    else if (y_type == I8_F16) i8_linear<I8_F16>(A, (hipStream_t)stream);
    else i8_linear<I8_BF16>(A, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}

template <int X>
static void i8_float(const I8Args& A, const void* x, int64_t ldx, int64_t inner, int y_type, hipStream_t stream)
{
    constexpr int size = (int)sizeof(typename I8Type<X>::T);
    if (y_type == I8_F32) i8_short<X, I8_F32>(A, x, ldx, inner, size, stream);
    else if (y_type == I8_F16) i8_short<X, I8_F16>(A, x, ldx, inner, size, stream);
    else i8_short<X, I8_BF16>(A, x, ldx, inner, size, stream);
}

extern "C" int64_t hrf_linear_int8_workspace_bytes(int64_t rows, int64_t cols, int64_t inner)
{
    if (rows <= 0 || cols <= 0 || inner < 1 || inner > HRF_INT8_MAX_INNER) return 0;
    return i8_is_short(rows, cols, i8_padded(inner)) ? 0 : rows * i8_padded(inner) + ((rows * 4 + 15) & ~(int64_t)15);
}

extern "C" int hrf_linear_int8_float(const void* x, int x_type, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias,
                                     int64_t rows, int64_t cols, int64_t inner, void* y, int y_type, int64_t ldy, int relu, void* workspace,
                                     hrf_stream_t stream)
{
    HRF_CHECK_ARG(x_type >= I8_F32 && x_type <= I8_BF16, "x_type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    HRF_CHECK_ARG(inner >= 1 && inner <= HRF_INT8_MAX_INNER, "bad sizes");
    const int64_t need = hrf_linear_int8_workspace_bytes(rows, cols, inner), padded = i8_padded(inner);
    int rc = i8_check(__func__, (const void*)16, padded, (const float*)16, w, ldw, w_scale, rows, cols, padded, y, y_type, ldy);
    if (rc || rows == 0 || cols == 0) return rc;
    HRF_CHECK_ARG(x, "NULL argument");
    HRF_CHECK_ARG(ldx >= inner || rows == 1, "a row stride is shorter than the row");
    if (need > 0) {
        HRF_CHECK_ARG(workspace && ((uintptr_t)workspace & 15u) == 0, "the workspace must begin at a multiple of 16 bytes");
        float* const scale = (float*)((int8_t*)workspace + rows * padded);
        rc = hrf_quantize_rows_int8(x, x_type, rows, inner, ldx, (int8_t*)workspace, padded, scale, stream);
        return rc ? rc : hrf_linear_int8((const int8_t*)workspace, padded, scale, w, ldw, w_scale, bias, rows, cols, padded, y, y_type, ldy, relu, stream);
    }
    I8Args A;
    A.x = nullptr; A.w = w; A.sx = nullptr; A.sw = w_scale; A.bias = bias; A.y = y; A.ldx = 0; A.ldw = ldw; A.ldy = ldy;
    A.rows = (int)rows; A.cols = (int)cols; A.inner = (int)padded; A.relu = relu;
    if (x_type == I8_F32) i8_float<I8_F32>(A, x, ldx, inner, y_type, (hipStream_t)stream);
    else if (x_type == I8_F16) i8_float<I8_F16>(A, x, ldx, inner, y_type, (hipStream_t)stream);
    else i8_float<I8_BF16>(A, x, ldx, inner, y_type, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}
