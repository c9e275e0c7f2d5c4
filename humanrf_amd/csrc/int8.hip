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
// One workgroup a row. A row that is not finite gets a scale that is not, and codes 0: its outputs are NaN.
template <int K>
__global__ __launch_bounds__(256) void k_quantize_rows(const typename I8Type<K>::T* __restrict__ x, int64_t cols, int64_t ldx,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale)
{
    __shared__ uint32_t s_max[4];
    x += (int64_t)blockIdx.x * ldx;
    q += (int64_t)blockIdx.x * ldq;
    uint32_t top = 0;       // of |x| as integers: the order of the values, NaN on top
    for (int64_t k = threadIdx.x; k < cols; k += 256) top = max(top, __float_as_uint(I8Type<K>::up(x[k])) & 0x7fffffffu);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    const bool finite = top < 0x7f800000u;
    const float amax = __uint_as_float(max(top, 0x04000000u));      // 2^-119: 127 / amax stays finite, a row of zeros gives zeros
    const float inverse = finite ? 127.0f / amax : 0.0f;
    if (threadIdx.x == 0) scale[blockIdx.x] = amax * (1.0f / 127.0f);
    for (int64_t k = threadIdx.x; k < ldq; k += 256)
        q[k] = k < cols && finite ? (int8_t)(int)rintf(I8Type<K>::up(x[k]) * inverse) : (int8_t)0;
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

// Rows of 64 bytes (inner <= 64): one instruction's k. A wavefront keeps the fragments of 64 channels in registers and walks over blocks of
// 16 tokens, whose operands come straight from memory.
template <int K>
__global__ __launch_bounds__(256) void k_linear_i8_short(const I8Args A)
{
    typedef typename I8Type<K>::T T;
    const int lane = threadIdx.x & 63;
    const int waves = (int)gridDim.x * 4, wave = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    const int n0 = (int)blockIdx.y * 64;
    const bool has_bias = A.bias != nullptr, relu = A.relu != 0;
    i8_v4 fw[4];
    float sw[4][4], bias[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int row = min(n0 + a * 16 + (lane & 15), A.cols - 1);
        fw[a] = *(const i8_v4*)(A.w + (int64_t)row * A.ldw + (lane >> 4) * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int n = min(n0 + a * 16 + (lane >> 4) * 4 + k, A.cols - 1);
            sw[a][k] = A.sw[n];
            bias[a][k] = has_bias ? A.bias[n] : 0.0f;
        }
    }
    const int blocks = (A.rows + 15) / 16;
    for (int blk = wave; blk < blocks; blk += waves) {
        const int m = blk * 16 + (lane & 15), row = min(m, A.rows - 1);
        const i8_v4 fx = *(const i8_v4*)(A.x + (int64_t)row * A.ldx + (lane >> 4) * 16);
        const float sx = A.sx[row];
        T* const y = (T*)A.y + (int64_t)row * A.ldy;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const i8_v4 acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[a], fx, i8_v4{0, 0, 0, 0}, 0, 0, 0);
            const int n = n0 + a * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (m < A.rows && n + k < A.cols) y[n + k] = i8_finish<K>(acc[k], sx, sw[a][k], bias[a][k], has_bias, relu);
        }
    }
}

template <int K>
static void i8_quantize(const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, hipStream_t stream)
{
    hipLaunchKernelGGL(k_quantize_rows<K>, dim3((unsigned)rows), dim3(256), 0, stream, (const typename I8Type<K>::T*)x, cols, ldx, q, ldq, scale);
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

template <int K>
static void i8_linear(const I8Args& A, hipStream_t stream)
{
    if (A.inner == 64) {
        const int64_t waves = ((int64_t)A.rows + 15) / 16;
        const unsigned blocks = (unsigned)std::min<int64_t>((waves + 3) / 4, 2048);
        hipLaunchKernelGGL((k_linear_i8_short<K>), dim3(blocks, (unsigned)((A.cols + 63) / 64)), dim3(256), 0, stream, A);
        return;
    }
    const int64_t large = (int64_t)((A.rows + 255) / 256) * ((A.cols + 255) / 256);
    if (large >= 200) hipLaunchKernelGGL((k_linear_i8<K, 4, 4>), dim3((unsigned)large), dim3(256), 0, stream, A);
    else {
        const int64_t tiles = (int64_t)((A.rows + 127) / 128) * ((A.cols + 127) / 128);
        hipLaunchKernelGGL((k_linear_i8<K, 2, 2>), dim3((unsigned)tiles), dim3(256), 0, stream, A);
    }
}

extern "C" int hrf_linear_int8(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                               const float* bias, int64_t rows, int64_t cols, int64_t inner, void* y, int y_type, int64_t ldy, int relu,
                               hrf_stream_t stream)
{
    HRF_CHECK_ARG(y_type >= I8_F32 && y_type <= I8_BF16, "y_type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
    HRF_CHECK_ARG(rows >= 0 && rows < ((int64_t)1 << 31) - 256 && cols >= 0 && cols < ((int64_t)1 << 31) - 256, "bad sizes");
    HRF_CHECK_ARG(inner >= 64 && inner <= HRF_INT8_MAX_INNER + 1 && inner == i8_padded(inner), "inner must be a padded length (hrf_int8_padded)");
    if (rows == 0 || cols == 0) return 0;
    HRF_CHECK_ARG(x && x_scale && w && w_scale && y, "NULL argument");
    HRF_CHECK_ARG((ldx >= inner || rows == 1) && (ldw >= inner || cols == 1) && (ldy >= cols || rows == 1), "a row stride is shorter than the row");
    HRF_CHECK_ARG((((uintptr_t)x | (uintptr_t)w) & 15u) == 0 && ((ldx | ldw) & 15) == 0, "x and w and their rows must begin at multiples of 16 bytes");
    HRF_CHECK_ARG(ldx < HRF_INT8_MAX_STRIDE && ldw < HRF_INT8_MAX_STRIDE, "rows are too far apart");
    HRF_CHECK_ARG(((rows + 127) / 128) * ((cols + 127) / 128) < ((int64_t)1 << 31) && cols <= 64 * 65535, "too many tiles");
    I8Args A;
    A.x = x; A.w = w; A.sx = x_scale; A.sw = w_scale; A.bias = bias; A.y = y; A.ldx = ldx; A.ldw = ldw; A.ldy = ldy;
    A.rows = (int)rows; A.cols = (int)cols; A.inner = (int)inner; A.relu = relu;
    if (y_type == I8_F32) i8_linear<I8_F32>(A, (hipStream_t)stream);
    else if (y_type == I8_F16) i8_linear<I8_F16>(A, (hipStream_t)stream);
    else i8_linear<I8_BF16>(A, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}
