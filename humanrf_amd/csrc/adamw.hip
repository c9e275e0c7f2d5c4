// AdamW (decoupled weight decay) over many tensors in one launch, moments in 32 or in 8 bits, and the global norm of their gradients.
//
// Per element, t = steps + 1, G = grad * f with f = min(1, max_norm / (norm + 1e-6)) / (grad_scale * loss scale):
//   m <- m + (G - m)(1 - b1)      v <- v b2 + (1 - b2) G G
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// every operation one fp32 rounding (built without contraction); what depends on t alone is computed in fp64 and rounded once.
//
// 8-bit states: m and r = sqrt(v) (half the exponent range of v) as e4m3 codes times one fp32 scale for every 256 values of a tensor,
// amax / 448. A code is the e4m3 value below or above |x| 448 / amax, above with the probability of the remainder (16 bits of a
// counter-based hash of seed, step and position): an average whose step is under half a code gap would never move under rounding to
// nearest -- a table entry without gradients would keep its first moment for ever and drift. r > 0 keeps a code > 0, so that a
// parameter with a first moment never divides by eps alone.
//
// Both passes stream: 28 B a parameter with fp32 p, g, m, v (bound by HBM), 16.06 B with 8-bit states.
#include "hrf_common.h"
#include <cmath>

#define AW_TILE 2048    // elements of one tensor that a workgroup of 256 works on at a time: two times four per thread
#define AW_BLOCK 256    // values that share a scale: one wavefront's four per lane
#define AW_NORM_BLOCKS 1024

typedef float aw_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t aw_u2 __attribute__((ext_vector_type(2)));

enum { AW_F32 = 0, AW_F16 = 1, AW_BF16 = 2 };

struct AwConst {
    double lr, beta1, beta2;
    float one_minus_b1, b2, one_minus_b2, eps;
    double max_norm;            // <= 0: no clipping
    double inv_grad_scale;
    const float* lr_dev;
    double weight_decay;
    const float* norm;
    const int32_t* flags;
    hrf_grad_scaler* scaler;
    uint32_t seed;
    int zero_grad;
};

__device__ __forceinline__ float aw_widen16(uint32_t h, bool bf16)
{
    return bf16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
__device__ __forceinline__ uint32_t aw_narrow16(float x, bool bf16)   // round to nearest even, as a copy to the type does
{
    return bf16 ? (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x) : (uint32_t)__half_as_ushort(__float2half_rn(x));
}

// Four consecutive values of a tensor of `kind`; `full`: all four are there and the address is a multiple of the access.
__device__ __forceinline__ void aw_load4(const void* base, int64_t i, int64_t n, int kind, bool full, float out[4])
{
    if (kind == AW_F32) {
        const float* p = (const float*)base + i;
        if (full) {
            const aw_f4 x = __builtin_nontemporal_load((const aw_f4*)p);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = x[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = i + k < n ? p[k] : 0.0f;
        }
    } else {
        const bool bf = kind == AW_BF16;
        const uint16_t* p = (const uint16_t*)base + i;
        if (full) {
            const aw_u2 x = __builtin_nontemporal_load((const aw_u2*)p);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = aw_widen16((x[k >> 1] >> (16 * (k & 1))) & 0xffffu, bf);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = i + k < n ? aw_widen16(p[k], bf) : 0.0f;
        }
    }
}

__device__ __forceinline__ void aw_store4(void* base, int64_t i, int64_t n, int kind, bool full, const float in[4], bool keep)
{
    if (kind == AW_F32) {
        float* p = (float*)base + i;
        if (full) __builtin_nontemporal_store(aw_f4{in[0], in[1], in[2], in[3]}, (aw_f4*)p);
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k) if (i + k < n) p[k] = in[k];
        }
    } else {
        const bool bf = kind == AW_BF16;
        uint16_t* p = (uint16_t*)base + i;
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = aw_narrow16(in[k], bf);
        if (full) {
            const aw_u2 x = {h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
            if (keep) *(aw_u2*)p = x;     // (the 16-bit copy is what the next forward pass reads: it stays cacheable)
            else __builtin_nontemporal_store(x, (aw_u2*)p);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) if (i + k < n) p[k] = (uint16_t)h[k];
        }
    }
}

__device__ __forceinline__ double aw_pow(double b, int32_t t)   // b^t by squaring: relative error of some 1e-15
{
    double r = 1.0;
    for (; t > 0; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// fp8 conversions of exactly representable values
__device__ __forceinline__ void aw_decode4(uint32_t codes, float scale, float out[4])
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    out[0] = lo[0] * scale; out[1] = lo[1] * scale; out[2] = hi[0] * scale; out[3] = hi[1] * scale;
}

__device__ __forceinline__ uint32_t aw_wave_max(uint32_t x)     // of values whose order as integers is theirs (|x|; NaN on top)
{
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, s));
    return x;
}

// amax of a block -> stored scale and the factor of the codes. Under 2^-100 the block is zeros (448 / amax would overflow soon after);
// inf or NaN in a block makes the scale and with it the whole block non-finite: seen, not hidden.
__device__ __forceinline__ void aw_scale(uint32_t amax_bits, float& scale, float& inverse)
{
    const float amax = __uint_as_float(amax_bits);
    if (amax < 0x1p-100f) { scale = 0.0f; inverse = 0.0f; return; }
    scale = amax * (1.0f / 448.0f);
    inverse = 448.0f / amax;
}

__device__ __forceinline__ float aw_round_e4m3(float ax, float inverse, uint32_t random16, bool floor)
{
    const float t = fminf(ax * inverse, 448.0f);
    // below 2^-6 e4m3 values are 2^-9 apart, which is the gap of the binade [2^-6, 2^-5): move the value there and back
    const float low = t < 0x1p-6f ? 0x1p-6f : 0.0f;
    const uint32_t bits = (__float_as_uint(t + low) + (random16 << 4)) & 0xfff00000u;   // 3 of 23 mantissa bits stay
    float q = fminf(__uint_as_float(bits) - low, 448.0f);
    if (floor && t > 0.0f) q = fmaxf(q, 0x1p-9f);
    return q;
}

__device__ __forceinline__ uint32_t aw_encode4(const float q[4])
{
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
}

struct AwStep { float factor, decay, step_size, inv_bc2; };

template <int kBits>
__global__ __launch_bounds__(256) void k_adamw(const hrf_adamw_tensor* __restrict__ tensors, const int32_t* __restrict__ tile_tensor,
                                               int num_tiles, int count, void* __restrict__ exp_avg, void* __restrict__ second,
                                               float* __restrict__ exp_avg_scale, float* __restrict__ second_scale, int32_t* ctl,
                                               const AwConst C)
{
    __shared__ int s_last;
    double inv = C.inv_grad_scale, lr = C.lr;
    if (C.scaler) inv /= (double)C.scaler->scale;
    if (C.lr_dev) lr = (double)*C.lr_dev;
    bool skip = C.flags && C.flags[0] != 0;
    if (C.norm) {
        const float norm = *C.norm;
        if (!(norm <= 3.402823466e38f)) skip = true;
        else if (C.max_norm > 0.0) inv *= fmin(1.0, C.max_norm / ((double)norm + 1e-6));
    }
    AwStep S;
    S.factor = (float)inv;
    int32_t known = -1;
    double known_lr = 0.0, known_decay = 0.0;
    uint32_t step_seed = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
        const int which = tile_tensor[tile];
        const hrf_adamw_tensor T = tensors[which];
        if (!T.grad) continue;          // no gradient this time: value, moments and step count stay
        const int pk = T.kind & 3, gk = (T.kind >> 2) & 3, ck = (T.kind >> 4) & 3;
        const int64_t begin = (int64_t)(tile - T.first_tile) * AW_TILE;
        const uintptr_t align = ((uintptr_t)T.param & (pk == AW_F32 ? 15u : 7u)) | ((uintptr_t)T.grad & (gk == AW_F32 ? 15u : 7u)) |
                                ((uintptr_t)T.copy & 7u);
        float p[2][4], g[2][4], m[2][4], r[2][4];
        bool full[2];
        int64_t at[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            at[u] = begin + u * 1024 + (int64_t)threadIdx.x * 4;
            full[u] = align == 0 && at[u] + 4 <= T.n;
        }
        if (skip) {
            if (C.zero_grad) {
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 2; ++u) aw_store4(T.grad, at[u], T.n, gk, full[u], zero, false);
            }
            continue;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (begin + u * 1024 + (int64_t)(threadIdx.x & 192) * 4 >= T.n) continue;   // (whole wavefronts: block-uniform)
            aw_load4(T.grad, at[u], T.n, gk, full[u], g[u]);
            aw_load4(T.param, at[u], T.n, pk, full[u], p[u]);
            const int64_t s = T.base + at[u];
            if (kBits == 32) {
                const aw_f4 mv = __builtin_nontemporal_load((const aw_f4*)((const float*)exp_avg + s));
                const aw_f4 vv = __builtin_nontemporal_load((const aw_f4*)((const float*)second + s));
#pragma unroll
                for (int k = 0; k < 4; ++k) { m[u][k] = mv[k]; r[u][k] = vv[k]; }
            } else {
                const int64_t b = s / AW_BLOCK;
                const uint32_t mc = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)exp_avg + s));
                const uint32_t rc = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)second + s));
                aw_decode4(mc, exp_avg_scale[b], m[u]);
                aw_decode4(rc, second_scale[b], r[u]);
            }
        }
        const int32_t t = ctl[4 + which] + 1;
        if (t != known || T.lr_scale != known_lr || T.decay_scale != known_decay) {
            known = t;
            known_lr = T.lr_scale;
            known_decay = T.decay_scale;
            S.decay = (float)(1.0 - (lr * T.lr_scale) * (C.weight_decay * T.decay_scale));
            S.step_size = (float)((lr * T.lr_scale) / (1.0 - aw_pow(C.beta1, t)));
            S.inv_bc2 = (float)(1.0 / sqrt(1.0 - aw_pow(C.beta2, t)));
            step_seed = hrf_mix32(C.seed ^ hrf_mix32((uint32_t)t));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (begin + u * 1024 + (int64_t)(threadIdx.x & 192) * 4 >= T.n) continue;
            float root[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float G = g[u][k] * S.factor;
                const float mk = m[u][k] + (G - m[u][k]) * C.one_minus_b1;
                const float vk = (kBits == 32 ? r[u][k] : r[u][k] * r[u][k]) * C.b2 + (G * C.one_minus_b2) * G;
                root[k] = sqrtf(vk);
                const float den = root[k] * S.inv_bc2 + C.eps;
                p[u][k] = p[u][k] * S.decay - (mk / den) * S.step_size;
                m[u][k] = mk;
                r[u][k] = vk;
            }
            aw_store4(T.param, at[u], T.n, pk, full[u], p[u], false);
            if (T.copy) aw_store4(T.copy, at[u], T.n, ck, full[u], p[u], true);
            if (C.zero_grad) {
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                aw_store4(T.grad, at[u], T.n, gk, full[u], zero, false);
            }
            const int64_t s = T.base + at[u];
            if (kBits == 32) {
                // (the states are padded to whole blocks: the last ones of a tensor are written too, zero in, zero out)
                __builtin_nontemporal_store(aw_f4{m[u][0], m[u][1], m[u][2], m[u][3]}, (aw_f4*)((float*)exp_avg + s));
                __builtin_nontemporal_store(aw_f4{r[u][0], r[u][1], r[u][2], r[u][3]}, (aw_f4*)((float*)second + s));
            } else {
                uint32_t am = 0, ar = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    am = max(am, __float_as_uint(m[u][k]) & 0x7fffffffu);
                    ar = max(ar, __float_as_uint(root[k]) & 0x7fffffffu);
                }
                am = aw_wave_max(am);
                ar = aw_wave_max(ar);
                float sm, im, sr, ir;
                aw_scale(am, sm, im);
                aw_scale(ar, sr, ir);
                float qm[4], qr[4];
                const uint32_t hi = hrf_mix32((uint32_t)((uint64_t)s >> 32));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t h = hrf_mix32(((uint32_t)s + k) ^ step_seed ^ hi);
                    qm[k] = copysignf(aw_round_e4m3(fabsf(m[u][k]), im, h & 0xffffu, false), m[u][k]);
                    qr[k] = aw_round_e4m3(root[k], ir, h >> 16, true);
                }
                __builtin_nontemporal_store(aw_encode4(qm), (uint32_t*)((uint8_t*)exp_avg + s));
                __builtin_nontemporal_store(aw_encode4(qr), (uint32_t*)((uint8_t*)second + s));
                if ((threadIdx.x & 63) == 0) {
                    exp_avg_scale[s / AW_BLOCK] = sm;
                    second_scale[s / AW_BLOCK] = sr;
                }
            }
        }
    }
    // The last workgroup to get here advances the step counts and the loss scale. Nothing but values read above (and consumed before the
    // barrier) is overwritten, and only the next launch reads what is written: a relaxed counter is enough.
    __syncthreads();
    if (threadIdx.x == 0) s_last = __hip_atomic_fetch_add(&ctl[0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    if (!s_last) return;
    if (!skip)
        for (int k = threadIdx.x; k < count; k += blockDim.x)
            if (tensors[k].grad) ctl[4 + k] += 1;
    if (threadIdx.x == 0) {
        if (skip) ctl[1] += 1;
        if (C.scaler) {     // torch.amp.GradScaler.update()
            if (skip) { C.scaler->scale *= C.scaler->backoff_factor; C.scaler->growth_tracker = 0; }
            else if (C.scaler->growth_tracker + 1 >= C.scaler->growth_interval) {
                C.scaler->scale *= C.scaler->growth_factor;
                C.scaler->growth_tracker = 0;
            } else C.scaler->growth_tracker += 1;
        }
        ctl[0] = 0;
    }
}

// Sum of squares in 64 bits (no overflow, and the same value in any order to 1e-16): every workgroup's sum into `partial`, the last
// workgroup adds them in the order of their numbers, so that the result does not depend on which finished when.
__global__ __launch_bounds__(256) void k_grad_norm(const hrf_adamw_tensor* __restrict__ tensors, const int32_t* __restrict__ tile_tensor,
                                                   int num_tiles, double* __restrict__ partial, int32_t* ticket, double inv_grad_scale,
                                                   const hrf_grad_scaler* __restrict__ scaler, float* __restrict__ out)
{
    __shared__ double s_sum[4];
    __shared__ int s_last;
    double sum = 0.0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
        const hrf_adamw_tensor T = tensors[tile_tensor[tile]];
        if (!T.grad) continue;
        const int gk = (T.kind >> 2) & 3;
        const int64_t begin = (int64_t)(tile - T.first_tile) * AW_TILE;
        const bool aligned = ((uintptr_t)T.grad & (gk == AW_F32 ? 15u : 7u)) == 0;
        float g[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t at = begin + u * 1024 + (int64_t)threadIdx.x * 4;
            aw_load4(T.grad, at, T.n, gk, aligned && at + 4 <= T.n, g[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += (double)g[u][k] * (double)g[u][k];
    }
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
        if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
        __syncthreads();
        const double total = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        if (pass == 1) {
            if (threadIdx.x == 0) {
                double inv = inv_grad_scale;
                if (scaler) inv /= (double)scaler->scale;
                *out = (float)(sqrt(total) * inv);
                *ticket = 0;
            }
            return;
        }
        if (threadIdx.x == 0) {
            __hip_atomic_store(&partial[blockIdx.x], total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        }
        __syncthreads();
        if (!s_last) return;
        sum = 0.0;
        for (int k = threadIdx.x; k < (int)gridDim.x; k += blockDim.x)
            sum += __hip_atomic_load(&partial[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

static bool aw_scaled(double x) { return std::isfinite(x) && x > 0.0; }

extern "C" size_t hrf_adamw_workspace_bytes(void) { return sizeof(double) * AW_NORM_BLOCKS; }

extern "C" int hrf_adamw_multi(const hrf_adamw_tensor* tensors, const int32_t* tile_tensor, int num_tiles, int count, int state_bits,
                               void* exp_avg, void* second, float* exp_avg_scale, float* second_scale, int32_t* ctl, double lr,
                               const float* lr_dev, double beta1, double beta2, double eps, double weight_decay, double grad_scale,
                               double max_norm, const float* norm, const int32_t* flags, hrf_grad_scaler* scaler, uint32_t seed,
                               int zero_grad, hrf_stream_t stream)
{
    HRF_CHECK_ARG(num_tiles >= 0 && count >= 0, "bad counts");
    HRF_CHECK_ARG(state_bits == 8 || state_bits == 32, "states are held in 8 or in 32 bits");
    HRF_CHECK_ARG(std::isfinite(lr) && lr >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 &&
                  std::isfinite(weight_decay) && weight_decay >= 0.0 && aw_scaled(grad_scale), "bad hyper-parameters");
    HRF_CHECK_ARG(std::isfinite(eps) && (float)eps >= 1.17549435e-38f, "eps has to be a positive normal fp32 number");
    HRF_CHECK_ARG(!(max_norm > 0.0) || norm, "clipping needs the norm of the gradients");
    if (num_tiles == 0) return 0;
    HRF_CHECK_ARG(tensors && tile_tensor && exp_avg && second && ctl, "NULL argument");
    HRF_CHECK_ARG(state_bits == 32 || (exp_avg_scale && second_scale), "8-bit states need their scales");
    AwConst C;
    C.lr = lr; C.beta1 = beta1; C.beta2 = beta2;
    C.one_minus_b1 = (float)(1.0 - beta1); C.b2 = (float)beta2; C.one_minus_b2 = (float)(1.0 - beta2); C.eps = (float)eps;
    C.max_norm = max_norm; C.inv_grad_scale = 1.0 / grad_scale; C.lr_dev = lr_dev; C.weight_decay = weight_decay;
    C.norm = norm; C.flags = flags; C.scaler = scaler; C.seed = seed; C.zero_grad = zero_grad;
    const unsigned blocks = num_tiles < 2048 ? (unsigned)num_tiles : 2048u;
    if (state_bits == 32)
        hipLaunchKernelGGL(k_adamw<32>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, count, exp_avg,
                           second, nullptr, nullptr, ctl, C);
    else
        hipLaunchKernelGGL(k_adamw<8>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, count, exp_avg,
                           second, exp_avg_scale, second_scale, ctl, C);
    HRF_CHECK_LAUNCH();
    return 0;
}

extern "C" int hrf_grad_norm_multi(const hrf_adamw_tensor* tensors, const int32_t* tile_tensor, int num_tiles, double grad_scale,
                                   const hrf_grad_scaler* scaler, int32_t* ctl, void* workspace, float* out, hrf_stream_t stream)
{
    HRF_CHECK_ARG(num_tiles >= 0 && aw_scaled(grad_scale), "bad counts / scale");
    HRF_CHECK_ARG(ctl && workspace && out && (num_tiles == 0 || (tensors && tile_tensor)), "NULL argument");
    const unsigned blocks = num_tiles < 1 ? 1u : num_tiles < AW_NORM_BLOCKS ? (unsigned)num_tiles : (unsigned)AW_NORM_BLOCKS;
    hipLaunchKernelGGL(k_grad_norm, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, (double*)workspace,
                       ctl + 2, 1.0 / grad_scale, scaler, out);
    HRF_CHECK_LAUNCH();
    return 0;
}
