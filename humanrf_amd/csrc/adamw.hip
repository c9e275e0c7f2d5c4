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
// Both passes stream: 28 B a parameter with fp32 p, g, m, v, 16.06 B with 8-bit states. On MI355X, where a copy of 4 GiB reads and writes
// 5.0 TB/s: 39 M fp32 parameters and their fp16 copy 189 us (6.2 TB/s) with 32-bit states, bound by HBM, and 124 us (5.7 TB/s) with 8-bit
// ones, whose 93 vector instructions an element keep the vector unit busy 78 % of that time; the norm of 240 M fp32 gradients 162 us
// (5.9 TB/s).
#include "hrf_common.h"
#include <algorithm>
#include <cmath>

#define AW_TILE 2048    // elements of one tensor that a workgroup of 256 works on at a time: two times four per thread
#define AW_BLOCK 256    // values that share a scale: one wavefront's four per lane
#define AW_NORM_BLOCKS 2048

typedef float aw_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t aw_u2 __attribute__((ext_vector_type(2)));
// the same at any address of its values (unaligned accesses are the hardware's)
typedef float aw_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t aw_u2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t aw_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t aw_u4u __attribute__((ext_vector_type(4), aligned(2)));

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

// Pointers that come out of a descriptor are generic to the compiler; they are typed as global so that the streams are global_load /
// global_store and not flat accesses.
#define AW_GLOBAL __attribute__((address_space(1)))

// Four consecutive values of a tensor of type K. kFull: all four are there; otherwise those below n, one by one.
template <int K, bool kFull>
__device__ __forceinline__ void aw_load4(const void* base, int64_t i, int64_t n, float out[4])
{
    if (K == AW_F32) {
        const AW_GLOBAL float* p = (const AW_GLOBAL float*)base + i;
        if (kFull) {
            const aw_f4 x = __builtin_nontemporal_load((const AW_GLOBAL aw_f4u*)p);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = x[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = i + k < n ? p[k] : 0.0f;
        }
    } else {
        const AW_GLOBAL uint16_t* p = (const AW_GLOBAL uint16_t*)base + i;
        if (kFull) {
            const aw_u2 x = __builtin_nontemporal_load((const AW_GLOBAL aw_u2u*)p);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = aw_widen16((x[k >> 1] >> (16 * (k & 1))) & 0xffffu, K == AW_BF16);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = i + k < n ? aw_widen16(p[k], K == AW_BF16) : 0.0f;
        }
    }
}

template <int K, bool kFull, bool kKeep>
__device__ __forceinline__ void aw_store4(void* base, int64_t i, int64_t n, const float in[4])
{
    if (K == AW_F32) {
        AW_GLOBAL float* p = (AW_GLOBAL float*)base + i;
        if (kFull) __builtin_nontemporal_store(aw_f4{in[0], in[1], in[2], in[3]}, (AW_GLOBAL aw_f4u*)p);
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k) if (i + k < n) p[k] = in[k];
        }
    } else {
        AW_GLOBAL uint16_t* p = (AW_GLOBAL uint16_t*)base + i;
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = aw_narrow16(in[k], K == AW_BF16);
        if (kFull) {
            const aw_u2 x = {h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
            if (kKeep) *(AW_GLOBAL aw_u2u*)p = x;     // (the 16-bit copy is what the next forward pass reads: it stays cacheable)
            else __builtin_nontemporal_store(x, (AW_GLOBAL aw_u2u*)p);
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

// Square root and quotient from the hardware's approximations (1 ulp) and one step of Newton's method, whose remainder an fma gives
// exactly: at most a few thousandths of an ulp over correct rounding, in 12 and 5 instructions where the library's take 18 and 11.
// Root: below 2^-100 the value is taken times 2^64 (the approximation flushes what is not normal); 0, inf and NaN are their own roots: a
// second moment beyond fp32 has no finite root, and the step that is divided by it is 0. Quotient: a denominator that is normal, inf or NaN.
__device__ __forceinline__ float aw_sqrt(float x)
{
    const bool tiny = x < 0x1p-100f;
    const float c = ldexpf(x, tiny ? 64 : 0);
    const float y = __builtin_amdgcn_rsqf(c), s = c * y;
    const float r = ldexpf(fmaf(fmaf(-s, s, c), 0.5f * y, s), tiny ? -32 : 0);
    return __builtin_amdgcn_classf(x, 0x180) ? r : x;       // positive, normal (0x100) or not (0x080)
}
__device__ __forceinline__ float aw_divide(float a, float b)
{
    const float y = __builtin_amdgcn_rcpf(b), q = a * y;
    return __builtin_amdgcn_div_fixupf(fmaf(fmaf(-q, b, a), y, q), b, a);
}

// fp8 conversions of exactly representable values
__device__ __forceinline__ void aw_decode4(uint32_t codes, float scale, float out[4])
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    out[0] = lo[0] * scale; out[1] = lo[1] * scale; out[2] = hi[0] * scale; out[3] = hi[1] * scale;
}

// Largest of a wavefront's values whose order as integers is theirs (|x|; NaN on top), the same in every lane: four steps inside rows
// of 16 lanes, two across them, all in the vector unit (no LDS permutes).
__device__ __forceinline__ uint32_t aw_wave_max(uint32_t x)
{
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true));    // row_shr:1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true));    // row_shr:2
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true));    // row_shr:4
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true));    // row_shr:8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));   // row_bcast:15 into rows 1 and 3
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));   // row_bcast:31 into rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
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
    const float t = ax * inverse;       // (up to a rounding over 448)
    // below 2^-6 e4m3 values are 2^-9 apart, which is the gap of the binade [2^-6, 2^-5): move the value there and back
    const float low = t < 0x1p-6f ? 0x1p-6f : 0.0f;
    const uint32_t bits = (__float_as_uint(t + low) + (random16 << 4)) & 0xfff00000u;   // 3 of 23 mantissa bits stay
    float q = __uint_as_float(min(bits, 0x43e00000u)) - low;      // at most 448, NaN too (its block's scale is not finite)
    if (floor && t > 0.0f) q = fmaxf(q, 0x1p-9f);
    return q;
}

__device__ __forceinline__ uint32_t aw_encode4(const float q[4])
{
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
}

// Whether the calling workgroup is the last of its launch (thread 0's answer; each workgroup asks once). Atomics on one address take
// 45-75 ns each, one after the other over the eight XCDs -- 90 us for 2048 workgroups on one counter --, so workgroups count in 32 groups on
// cache lines of their own and the last of a group counts in the root. The counters are zero again when the launch ends.
__device__ __forceinline__ bool aw_last(int32_t* tickets)
{
    const int group = blockIdx.x & (HRF_ADAMW_TICKETS - 1), groups = min((int)gridDim.x, HRF_ADAMW_TICKETS);
    const int members = ((int)gridDim.x - group + HRF_ADAMW_TICKETS - 1) / HRF_ADAMW_TICKETS;
    int32_t* own = tickets + 32 * (1 + group);
    if (__hip_atomic_fetch_add(own, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != members - 1) return false;
    __hip_atomic_store(own, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__hip_atomic_fetch_add(tickets, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != groups - 1) return false;
    __hip_atomic_store(tickets, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

struct AwStep { float factor, decay, step_size, inv_bc2; uint32_t seed; };

// One tile: all loads of both halves first, then the arithmetic, then the stores.
template <int kBits, int PK, int GK, bool kFull>
__device__ __forceinline__ void aw_tile(const hrf_adamw_tensor& T, int64_t begin, const AwConst& C, const AwStep& S, void* exp_avg,
                                        void* second, float* exp_avg_scale, float* second_scale)
{
    const int ck = (T.kind >> 4) & 3;
    float p[2][4], g[2][4], m[2][4], r[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t at = begin + u * 1024 + (int)threadIdx.x * 4, s = T.base + at;
        if (!kFull && begin + u * 1024 + (int)(threadIdx.x & 192) * 4 >= T.n) continue;      // (whole wavefronts)
        aw_load4<GK, kFull>(T.grad, at, T.n, g[u]);
        aw_load4<PK, kFull>(T.param, at, T.n, p[u]);
        if (kBits == 32) {
            const aw_f4 mv = __builtin_nontemporal_load((const aw_f4*)((const float*)exp_avg + s));
            const aw_f4 vv = __builtin_nontemporal_load((const aw_f4*)((const float*)second + s));
#pragma unroll
            for (int k = 0; k < 4; ++k) { m[u][k] = mv[k]; r[u][k] = vv[k]; }
        } else {
            const uint32_t mc = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)exp_avg + s));
            const uint32_t rc = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)second + s));
            aw_decode4(mc, exp_avg_scale[s / AW_BLOCK], m[u]);
            aw_decode4(rc, second_scale[s / AW_BLOCK], r[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t at = begin + u * 1024 + (int)threadIdx.x * 4, s = T.base + at;
        if (!kFull && begin + u * 1024 + (int)(threadIdx.x & 192) * 4 >= T.n) continue;
        float root[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float G = g[u][k] * S.factor;
            const float mk = m[u][k] + (G - m[u][k]) * C.one_minus_b1;
            const float vk = (kBits == 32 ? r[u][k] : r[u][k] * r[u][k]) * C.b2 + (G * C.one_minus_b2) * G;
            root[k] = aw_sqrt(vk);
            const float den = root[k] * S.inv_bc2 + C.eps;
            p[u][k] = p[u][k] * S.decay - aw_divide(mk, den) * S.step_size;
            m[u][k] = mk;
            r[u][k] = vk;
        }
        aw_store4<PK, kFull, false>(T.param, at, T.n, p[u]);
        if (T.copy) {
            if (ck == AW_BF16) aw_store4<AW_BF16, kFull, true>(T.copy, at, T.n, p[u]);
            else aw_store4<AW_F16, kFull, true>(T.copy, at, T.n, p[u]);
        }
        if (C.zero_grad) {
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            aw_store4<GK, kFull, false>(T.grad, at, T.n, zero);
        }
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
            float sm, im, sr, ir;
            aw_scale(aw_wave_max(am), sm, im);
            aw_scale(aw_wave_max(ar), sr, ir);
            float qm[4], qr[4];
            // (a wavefront's block of 256 lies on one side of any multiple of 2^32)
            const uint32_t mixed = S.seed ^ hrf_mix32((uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)s >> 32)));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t h = hrf_mix32(((uint32_t)s + k) ^ mixed);
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

template <int GK>
__device__ __forceinline__ void aw_zero_tile(const hrf_adamw_tensor& T, int64_t begin)
{
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 2; ++u) aw_store4<GK, false, false>(T.grad, begin + u * 1024 + (int)threadIdx.x * 4, T.n, zero);
}

template <int kBits>
__global__ __launch_bounds__(256) void k_adamw(const hrf_adamw_tensor* __restrict__ tensors, const int32_t* __restrict__ tile_tensor,
                                               int num_tiles, int count, void* __restrict__ exp_avg, void* __restrict__ second,
                                               float* __restrict__ exp_avg_scale, float* __restrict__ second_scale, int32_t* ctl,
                                               int per, const AwConst C)
{
    __shared__ int s_last;
    const int tile_end = min(num_tiles, (int)(blockIdx.x + 1) * per);
    int which = num_tiles > 0 ? tile_tensor[blockIdx.x * per] : 0;
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
    for (int tile = blockIdx.x * per; tile < tile_end;) {
        const hrf_adamw_tensor T = tensors[which];
        const int32_t t = ctl[HRF_ADAMW_CTL + which] + 1;
        const int64_t begin = (int64_t)(tile - T.first_tile) * AW_TILE;
        ++tile;
        if (tile < tile_end) which = tile_tensor[tile];     // (the next tile's tensor is on its way while this one is stepped)
        if (!T.grad) continue;          // no gradient this time: value, moments and step count stay
        const int gk = (T.kind >> 2) & 3;
        if (skip) {
            if (C.zero_grad) {
                if (gk == AW_F32) aw_zero_tile<AW_F32>(T, begin);
                else aw_zero_tile<AW_F16>(T, begin);        // (zero is zero in either 16-bit type)
            }
            continue;
        }
        if (t != known || T.lr_scale != known_lr || T.decay_scale != known_decay) {
            known = t;
            known_lr = T.lr_scale;
            known_decay = T.decay_scale;
            S.decay = (float)(1.0 - (lr * T.lr_scale) * (C.weight_decay * T.decay_scale));
            S.step_size = (float)((lr * T.lr_scale) / (1.0 - aw_pow(C.beta1, t)));
            S.inv_bc2 = (float)(1.0 / sqrt(1.0 - aw_pow(C.beta2, t)));
            S.seed = hrf_mix32(C.seed ^ hrf_mix32((uint32_t)t));
        }
        const bool full = begin + AW_TILE <= T.n;
#define AW_CASE(P, G)                                                                                        \
    case (P) | ((G) << 2):                                                                                   \
        if (full) aw_tile<kBits, P, G, true>(T, begin, C, S, exp_avg, second, exp_avg_scale, second_scale);  \
        else aw_tile<kBits, P, G, false>(T, begin, C, S, exp_avg, second, exp_avg_scale, second_scale);      \
        break;
        switch (T.kind & 15) {
            AW_CASE(AW_F32, AW_F32) AW_CASE(AW_F32, AW_F16) AW_CASE(AW_F32, AW_BF16)
            AW_CASE(AW_F16, AW_F32) AW_CASE(AW_F16, AW_F16) AW_CASE(AW_F16, AW_BF16)
            AW_CASE(AW_BF16, AW_F32) AW_CASE(AW_BF16, AW_F16) AW_CASE(AW_BF16, AW_BF16)
        }
#undef AW_CASE
    }
    // The last workgroup to get here advances the step counts and the loss scale. Nothing but values read above (and consumed before the
    // barrier) is overwritten, and only the next launch reads what is written: a relaxed counter is enough.
    __syncthreads();
    if (threadIdx.x == 0) s_last = aw_last(ctl + 32);
    __syncthreads();
    if (!s_last) return;
    if (!skip)
        for (int k = threadIdx.x; k < count; k += blockDim.x)
            if (tensors[k].grad) ctl[HRF_ADAMW_CTL + k] += 1;
    if (threadIdx.x == 0) {
        if (skip) ctl[0] += 1;
        if (C.scaler) {     // torch.amp.GradScaler.update()
            if (skip) { C.scaler->scale *= C.scaler->backoff_factor; C.scaler->growth_tracker = 0; }
            else if (C.scaler->growth_tracker + 1 >= C.scaler->growth_interval) {
                C.scaler->scale *= C.scaler->growth_factor;
                C.scaler->growth_tracker = 0;
            } else C.scaler->growth_tracker += 1;
        }
    }
}

template <int kThreads>
__device__ __forceinline__ double aw_block_sum(double sum)     // over the workgroup, in a fixed order, for thread 0
{
    __shared__ double s_sum[kThreads / 64];
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) total += s_sum[w];
    return total;
}

// Sum of squares in 64 bits: no overflow, and the same value in any order to 1e-16. 256 threads a tile; every workgroup's sum into `partial`,
// or, where there is one workgroup, the norm itself.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void k_grad_norm(const hrf_adamw_tensor* __restrict__ tensors, const int32_t* __restrict__ tile_tensor,
                                                   int num_tiles, double* __restrict__ partial, double inv_grad_scale,
                                                        const hrf_grad_scaler* __restrict__ scaler, float* __restrict__ out)
{
    double sum = 0.0;
    // (a wavefront's tile is a scalar: a vector's worth of descriptors costs a fifth of the bandwidth)
    const int thread = kThreads == 256 ? (int)threadIdx.x : (int)(threadIdx.x & 255), stride = kThreads == 256 ? (int)gridDim.x : kThreads / 256;
    const int first = kThreads == 256 ? (int)blockIdx.x : __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 8));
    int which = first < num_tiles ? tile_tensor[first] : 0;
    for (int tile = first; tile < num_tiles;) {
        const void* grad = tensors[which].grad;
        const int64_t n = tensors[which].n, begin = (int64_t)(tile - tensors[which].first_tile) * AW_TILE;
        const int gk = (tensors[which].kind >> 2) & 3;
        tile += stride;
        if (tile < num_tiles) which = tile_tensor[tile];
        if (!grad) continue;
        float g[8];
        if (begin + AW_TILE <= n) {
            if (gk == AW_F32) {
                const AW_GLOBAL aw_f4u* p = (const AW_GLOBAL aw_f4u*)((const float*)grad + begin) + thread;
                const aw_f4 x = p[0], y = p[256];
#pragma unroll
                for (int k = 0; k < 4; ++k) { g[k] = x[k]; g[4 + k] = y[k]; }
            } else {
                const aw_u4 x = *((const AW_GLOBAL aw_u4u*)((const uint16_t*)grad + begin) + thread);
#pragma unroll
                for (int k = 0; k < 8; ++k) g[k] = aw_widen16((x[k >> 1] >> (16 * (k & 1))) & 0xffffu, gk == AW_BF16);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t at = begin + u * 1024 + thread * 4;
                if (gk == AW_F32) aw_load4<AW_F32, false>(grad, at, n, g + 4 * u);
                else if (gk == AW_F16) aw_load4<AW_F16, false>(grad, at, n, g + 4 * u);
                else aw_load4<AW_BF16, false>(grad, at, n, g + 4 * u);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += (double)g[k] * (double)g[k];
    }
    sum = aw_block_sum<kThreads>(sum);
    if (threadIdx.x != 0) return;
    if (kThreads == 256) partial[blockIdx.x] = sum;
    else *out = (float)(sqrt(sum) * (scaler ? inv_grad_scale / (double)scaler->scale : inv_grad_scale));
}

// The workgroups' sums in the order of their numbers. (A launch of its own: letting the last workgroup of the first one do it takes a
// release fence in each of them, which holds back 2048 workgroups for 92 us where reading 156 MB takes 30.)
__global__ __launch_bounds__(256) void k_grad_norm_end(const double* __restrict__ partial, int blocks, double inv_grad_scale,
                                                       const hrf_grad_scaler* __restrict__ scaler, float* __restrict__ out)
{
    double sum = 0.0;
    for (int k = threadIdx.x; k < blocks; k += 256) sum += partial[k];
    sum = aw_block_sum<256>(sum);
    if (threadIdx.x == 0) *out = (float)(sqrt(sum) * (scaler ? inv_grad_scale / (double)scaler->scale : inv_grad_scale));
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
    HRF_CHECK_ARG(!scaler || norm || flags, "a loss scale needs the norm of the gradients or flags to see that they are finite");
    if (num_tiles == 0 && (count == 0 || !tensors)) return 0;
    HRF_CHECK_ARG(tensors && ctl && (num_tiles == 0 || (tile_tensor && exp_avg && second)), "NULL argument");
    HRF_CHECK_ARG(state_bits == 32 || num_tiles == 0 || (exp_avg_scale && second_scale), "8-bit states need their scales");
    HRF_CHECK_ARG((((uintptr_t)exp_avg | (uintptr_t)second) & 15u) == 0, "states must begin at multiples of 16 bytes");
    AwConst C;
    C.lr = lr; C.beta1 = beta1; C.beta2 = beta2;
    C.one_minus_b1 = (float)(1.0 - beta1); C.b2 = (float)beta2; C.one_minus_b2 = (float)(1.0 - beta2); C.eps = (float)eps;
    C.max_norm = max_norm; C.inv_grad_scale = 1.0 / grad_scale; C.lr_dev = lr_dev; C.weight_decay = weight_decay;
    C.norm = norm; C.flags = flags; C.scaler = scaler; C.seed = seed; C.zero_grad = zero_grad;
    // One tile per workgroup, so that the scheduler evens out the work: 39 M fp32 parameters with 32-bit states 191 us against 208 us with
    // 2048 workgroups striding over the tiles; 120 M bf16 ones 430 against 518. 8-bit states are near the vector unit's limit, and what a
    // workgroup computes once (the bias corrections, in fp64) counts: four neighbouring tiles each, where that leaves eight workgroups
    // for every CU. Calls timed by events: 240 M parameters 710 us against 738 with one tile each, 39 M 149 against 153.
    const int per = state_bits == 8 && num_tiles >= 4 * 2048 ? 4 : 1;
    const unsigned blocks = (unsigned)std::max(1, (num_tiles + per - 1) / per);    // (tensors without a value have a step count)
    if (state_bits == 32)
        hipLaunchKernelGGL(k_adamw<32>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, count, exp_avg,
                           second, nullptr, nullptr, ctl, per, C);
    else
        hipLaunchKernelGGL(k_adamw<8>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, count, exp_avg,
                           second, exp_avg_scale, second_scale, ctl, per, C);
    HRF_CHECK_LAUNCH();
    return 0;
}

extern "C" int hrf_grad_norm_multi(const hrf_adamw_tensor* tensors, const int32_t* tile_tensor, int num_tiles, double grad_scale,
                                   const hrf_grad_scaler* scaler, void* workspace, float* out, hrf_stream_t stream)
{
    HRF_CHECK_ARG(num_tiles >= 0 && aw_scaled(grad_scale), "bad counts / scale");
    HRF_CHECK_ARG(workspace && out && (num_tiles == 0 || (tensors && tile_tensor)), "NULL argument");
    // One workgroup up to 16 tiles: 8 tiles 3.4 us captured and 5.6 called against 4.2 and 8.6 for two launches, 16 tiles 4.6 / 5.6 against
    // 4.4 / 8.8, 32 tiles 7.0 / 7.0 against 4.3 / 8.7.
    if (num_tiles <= 16) {
        hipLaunchKernelGGL(k_grad_norm<1024>, dim3(1), dim3(1024), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, (double*)workspace,
                           1.0 / grad_scale, scaler, out);
    } else {
        const unsigned blocks = num_tiles < AW_NORM_BLOCKS ? (unsigned)num_tiles : (unsigned)AW_NORM_BLOCKS;
        hipLaunchKernelGGL(k_grad_norm<256>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tensors, tile_tensor, num_tiles, (double*)workspace,
                           1.0, nullptr, nullptr);
        hipLaunchKernelGGL(k_grad_norm_end, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)workspace, (int)blocks, 1.0 / grad_scale,
                           scaler, out);
    }
    HRF_CHECK_LAUNCH();
    return 0;
}
