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

// Tiles of BM tokens x BN channels, four wavefronts 2 x 2, 128 bytes of k a stage, two stages in LDS, filled by direct loads. A row's
// eight 16-byte chunks lie in LDS permuted by its number, so that 16 lanes that read the same chunk of 16 rows hit all banks.
template <int K, int BM, int BN>
__global__ __launch_bounds__(256) void k_linear_i8(const I8Args A)
{
    constexpr int MT = BM / 32, NT = BN / 32;       // 16 x 16 tiles of a wavefront
    __shared__ __align__(16) int8_t s_tile[2][(BM + BN) * 128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
    const int tiles_m = (A.rows + BM - 1) / BM;
    const int m0 = (blockIdx.x % tiles_m) * BM, n0 = (blockIdx.x / tiles_m) * BN;
    const int8_t* const xb = A.x + (int64_t)m0 * A.ldx;
    const int8_t* const wb = A.w + (int64_t)n0 * A.ldw;
    const int stage = min(128, A.inner);
    const int steps = A.inner / stage;
    const int r8 = lane >> 3, c8 = lane & 7;

    auto load = [&](int buf, int k0) {
#pragma unroll
        for (int i = 0; i < (BM + BN) / 32; ++i) {
            const int first = (i * 4 + wave) * 8;           // the wavefront's eight rows (wave-uniform)
            const int r = first + r8, chunk = c8 ^ (r & 7);
            const bool is_x = first < BM;
            const int row = is_x ? min(r, A.rows - 1 - m0) : min(r - BM, A.cols - 1 - n0);
            // (a row of 64 bytes has four chunks: the others are read twice and not used)
            const int8_t* src = (is_x ? xb + (int64_t)row * A.ldx : wb + (int64_t)row * A.ldw) + k0 + ((chunk * 16) & (stage - 1));
            __builtin_amdgcn_global_load_lds((const I8_GLOBAL void*)src, (I8_LDS void*)&s_tile[buf][first * 128], 16, 0, 0);
        }
    };
    i8_v4 acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[a][b] = i8_v4{0, 0, 0, 0};
    load(0, 0);
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < steps) load((s + 1) & 1, (s + 1) * stage);
        const int8_t* t = s_tile[s & 1];
        for (int kk = 0; kk < stage / 64; ++kk) {
            i8_v4 fx[MT], fw[NT];
            const int chunk = kk * 4 + (lane >> 4);
#pragma unroll
            for (int b = 0; b < MT; ++b) {
                const int r = wm * (BM / 2) + b * 16 + (lane & 15);
                fx[b] = *(const i8_v4*)(t + r * 128 + ((chunk ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const int r = BM + wn * (BN / 2) + a * 16 + (lane & 15);
                fw[a] = *(const i8_v4*)(t + r * 128 + ((chunk ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int b = 0; b < MT; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[a], fx[b], acc[a][b], 0, 0, 0);
        }
    }
    typedef typename I8Type<K>::T T;
#pragma unroll
    for (int b = 0; b < MT; ++b) {
        const int m = m0 + wm * (BM / 2) + b * 16 + (lane & 15);
        if (m >= A.rows) continue;
        const float sx = A.sx[m];
        T* y = (T*)A.y + (int64_t)m * A.ldy;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            const int n = n0 + wn * (BN / 2) + a * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n + k < A.cols)
                    y[n + k] = i8_finish<K>(acc[a][b][k], sx, A.sw[n + k], A.bias ? A.bias[n + k] : 0.0f, A.bias != nullptr, A.relu != 0);
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
    const int64_t tiles = (int64_t)((A.rows + 127) / 128) * ((A.cols + 127) / 128);
    hipLaunchKernelGGL((k_linear_i8<K, 128, 128>), dim3((unsigned)tiles), dim3(256), 0, stream, A);
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
    HRF_CHECK_ARG(((rows + 63) / 64) * ((cols + 63) / 64) < ((int64_t)1 << 31), "too many tiles");
    I8Args A;
    A.x = x; A.w = w; A.sx = x_scale; A.sw = w_scale; A.bias = bias; A.y = y; A.ldx = ldx; A.ldw = ldw; A.ldy = ldy;
    A.rows = (int)rows; A.cols = (int)cols; A.inner = (int)inner; A.relu = relu;
    if (y_type == I8_F32) i8_linear<I8_F32>(A, (hipStream_t)stream);
    else if (y_type == I8_F16) i8_linear<I8_F16>(A, (hipStream_t)stream);
    else i8_linear<I8_BF16>(A, (hipStream_t)stream);
    HRF_CHECK_LAUNCH();
    return 0;
}
