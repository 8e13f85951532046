// The AdamW step over many tensors, with moments in 32 bits or in 8 (cx_adamw_step), and the way between
// the 8-bit moments and their values (cx_adamw_states, cx_adamw_set_states).  Formulas and formats:
// include/comprex_gfx950.h.
//
// No product or sum below is contracted: the moments have the same bits whatever the compiler does
// around them, so an 8-bit code never depends on the build.  Where a fused multiply-add is wanted it is
// written out.
#include "cx_tensors.hpp"

#include <cmath>

#pragma clang fp contract(off)

namespace cx {

namespace {

constexpr int kBlock = 256;

// What depends on the step's count.
struct AdamwRates {
    float step;        // lr / (1 - beta1^t)
    float decay;       // lr * weight_decay
    float v_unit;      // 1 / sqrt(1 - beta2^t)
};

struct AdamwArgs {
    float beta1, rest1, beta2, rest2, eps, scale;   // rest = 1 - beta, rounded from 64 bits
    AdamwRates rates;
    const AdamwRates* device_rates;                 // replaces `rates` where the count lives on the device
    const float* coefs;
    int per_tensor;
    const int* skip;
};

__host__ __device__ inline AdamwRates rates_of(double lr, double beta1, double beta2, double weight_decay, double t) {
    AdamwRates r;
    r.step = (float)(lr / (1.0 - pow(beta1, t)));
    r.decay = (float)(lr * weight_decay);
    r.v_unit = (float)(1.0 / sqrt(1.0 - pow(beta2, t)));
    return r;
}

// The step's count on the device: one thread advances it and leaves the rates for the step's kernel.
__global__ void rates_kernel(int* count, long long step, const float* d_lr, double lr, double beta1, double beta2,
                             double weight_decay, const int* skip, AdamwRates* rates) {
    if (skip && *skip) return;
    if (count) step = ++*count;
    *rates = rates_of(d_lr ? (double)*d_lr : lr, beta1, beta2, weight_decay, (double)step);
}

// The moments of four elements; g already has its factor.
__device__ __forceinline__ void moments(Vec4<float> g, const AdamwArgs& a, Vec4<float>& m, Vec4<float>& v) {
    m = m * a.beta1 + g * a.rest1;
    v = v * a.beta2 + g * g * a.rest2;
}

__device__ __forceinline__ Vec4<float> weights(Vec4<float> w, Vec4<float> m, Vec4<float> v, const AdamwArgs& a,
                                               const AdamwRates& r) {
    for (int k = 0; k < 4; ++k) {
        const float below = __builtin_fmaf(__builtin_sqrtf(v[k]), r.v_unit, a.eps);
        w[k] -= __builtin_fmaf(r.decay, w[k], r.step * (m[k] / below));
    }
    return w;
}

template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kBlock) void adamw32_kernel(const Chunk* __restrict__ chunks, int first, GradArgs ga,
                                                         AdamwArgs a) {
    const Chunk c = chunks[first + blockIdx.x];
    const G* g = grad_of<G>(c, ga);
    if (!g || (a.skip && *a.skip)) return;
    const AdamwRates r = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    P* p = static_cast<P*>(c.param);
    float *pm = static_cast<float*>(c.m), *pv = static_cast<float*>(c.v);
    for (int i = threadIdx.x * 4; i < c.n; i += kBlock * 4) {
        const int k = c.n - i;
        const Vec4<float> x = to_float<G>(load_up_to4(g + i, k)) * f;
        Vec4<float> m = load_up_to4(pm + i, k), v = load_up_to4(pv + i, k);
        Vec4<float> w;
        if constexpr (MASTER) w = load_up_to4(c.master + i, k);
        else w = to_float<P>(load_up_to4(p + i, k));
        moments(x, a, m, v);
        w = weights(w, m, v, a, r);
        store_up_to4(pm + i, m, k);
        store_up_to4(pv + i, v, k);
        if constexpr (MASTER) store_up_to4(c.master + i, w, k);
        store_up_to4(p + i, from_float<P>(w), k);
    }
}

// ---- 8-bit moments ---------------------------------------------------------------------------
// A wave holds four blocks of 256 elements, 16 lanes a block (a row of the lane crossbar): lane r of a row
// has the elements j * 64 + r * 4 + 0..3, j = 0..3.  Each load of the wave then takes 256 contiguous bytes
// of fp32 from each block, and a block's maximum is 4 row rotations, not 6 steps over the wave, for 16
// elements a lane.

constexpr int kGroup = 4 * CX_STATE_BLOCK;       // elements of a wave's four blocks
constexpr float kTiny = 0x1p-100f;               // a block below is stored as zeros
constexpr float kVUnit = 0x1.ep-96f;             // V lies here before its bits are cut: exponent field 31, fraction 7/8
constexpr float kVBack = (float)(0x1p96 / 1.875);

__device__ __forceinline__ unsigned row_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));  // rotate the row by 8
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
    return x;
}

// The largest finite magnitude of a row's 64 x 4 values (floats of one sign order like their bits).
__device__ __forceinline__ float block_max(const Vec4<float> (&x)[4]) {
    unsigned top = 0;
    for (int j = 0; j < 4; ++j)
        for (int k = 0; k < 4; ++k) {
            const unsigned u = __float_as_uint(x[j][k]) & 0x7fffffffu;
            top = max(top, u < 0x7f800000u ? u : 0u);
        }
    return __uint_as_float(row_max(top));
}

__device__ __forceinline__ Vec4<float> m_value(unsigned codes, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return Vec4<float>{lo[0], lo[1], hi[0], hi[1]} * scale;
}
__device__ __forceinline__ Vec4<float> v_value(unsigned codes, float scale) {
    Vec4<float> x;
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(((codes >> (8 * k)) & 255u) << 20);
    return x * kVBack * scale;
}
__device__ __forceinline__ unsigned m_codes(Vec4<float> m, float inverse) {
    m = m * inverse;
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(m[0], m[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[2], m[3], u, true);
}
// The value's own exponent and upper fraction bits, after a scaling that leaves 5 bits of exponent: small
// values run into the format's subnormals as they do into those of fp32.  Rounded to nearest.
__device__ __forceinline__ unsigned v_codes(Vec4<float> v, float inverse) {
    const Vec4<float> y = v * inverse * kVUnit;
    unsigned u = 0;
    for (int k = 0; k < 4; ++k) {
        unsigned code = min((__float_as_uint(y[k]) + 0x80000u) >> 20, 255u);
        code = max(code, min(__float_as_uint(v[k]), 1u));  // above 0: never 0
        u |= code << (8 * k);
    }
    return u;
}

// Rounds the moments of a row's block and stores codes and scales; lane `r` of the row, n elements of the
// block there (at least one), `block` and the codes' base within the piece.
template <bool FULL>
__device__ __forceinline__ void store_states(const Vec4<float> (&m)[4], const Vec4<float> (&v)[4], unsigned char* pm,
                                             unsigned char* pv, float* sm, float* sv, int r, int n) {
    const float mt = block_max(m), vt = block_max(v);
    const bool m_kept = mt >= kTiny, v_kept = vt >= kTiny;
    const float m_inverse = m_kept ? 448.0f / mt : 0.0f, v_inverse = v_kept ? 1.0f / vt : 0.0f;
    if (!FULL && n <= 0) return;
    if (r == 0) {
        *sm = m_kept ? mt * (float)(1.0 / 448.0) : 0.0f;
        *sv = v_kept ? vt : 0.0f;
    }
    for (int j = 0; j < 4; ++j) {
        const int i = j * 64 + r * 4, k = FULL ? 4 : n - i;
        const unsigned mc = m_codes(m[j], m_inverse), vc = v_kept ? v_codes(v[j], v_inverse) : 0u;
        store_up_to4(pm + i, __builtin_bit_cast(Vec4<unsigned char>, mc), k);
        store_up_to4(pv + i, __builtin_bit_cast(Vec4<unsigned char>, vc), k);
    }
}

template <typename P, typename G, bool MASTER, bool FULL>
__device__ __forceinline__ void adamw8_group(const Chunk& c, const G* g, int at, int r, int n, int block,
                                             const AdamwArgs& a, const AdamwRates& rates, float f) {
    P* p = static_cast<P*>(c.param) + at;
    unsigned char *pm = static_cast<unsigned char*>(c.m) + at, *pv = static_cast<unsigned char*>(c.v) + at;
    g += at;
    const bool there = FULL || n > 0;
    const float sm = there ? c.m_scale[block] : 0.0f, sv = there ? c.v_scale[block] : 0.0f;
    Vec4<float> m[4], v[4];
    for (int j = 0; j < 4; ++j) {
        const int i = j * 64 + r * 4, k = FULL ? 4 : n - i;
        const Vec4<float> x = to_float<G>(load_up_to4(g + i, k)) * f;
        Vec4<float> w;
        if constexpr (MASTER) w = load_up_to4(c.master + at + i, k);
        else w = to_float<P>(load_up_to4(p + i, k));
        m[j] = m_value(__builtin_bit_cast(unsigned, load_up_to4(pm + i, k)), sm);
        v[j] = v_value(__builtin_bit_cast(unsigned, load_up_to4(pv + i, k)), sv);
        moments(x, a, m[j], v[j]);
        w = weights(w, m[j], v[j], a, rates);
        if constexpr (MASTER) store_up_to4(c.master + at + i, w, k);
        store_up_to4(p + i, from_float<P>(w), k);
    }
    store_states<FULL>(m, v, pm, pv, c.m_scale + block, c.v_scale + block, r, n);
}

template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kBlock) void adamw8_kernel(const Chunk* __restrict__ chunks, int first, GradArgs ga,
                                                        AdamwArgs a) {
    const Chunk c = chunks[first + blockIdx.x];
    const G* g = grad_of<G>(c, ga);
    if (!g || (a.skip && *a.skip)) return;
    const AdamwRates rates = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    const int row = (threadIdx.x & 63) >> 4, r = threadIdx.x & 15;
    for (int q = (threadIdx.x >> 6) * kGroup; q < c.n; q += kBlock / 64 * kGroup) {
        const int at = q + row * CX_STATE_BLOCK, block = at / CX_STATE_BLOCK;
        if (q + kGroup <= c.n) adamw8_group<P, G, MASTER, true>(c, g, at, r, CX_STATE_BLOCK, block, a, rates, f);
        else adamw8_group<P, G, MASTER, false>(c, g, at, r, c.n - at, block, a, rates, f);
    }
}

template <typename E>
__global__ __launch_bounds__(kBlock) void states_kernel(const Chunk* __restrict__ chunks, E* __restrict__ m_out,
                                                        E* __restrict__ v_out) {
    const Chunk c = chunks[blockIdx.x];
    const unsigned char *pm = static_cast<const unsigned char*>(c.m), *pv = static_cast<const unsigned char*>(c.v);
    for (int i = threadIdx.x * 4; i < c.n; i += kBlock * 4) {
        const int k = c.n - i, block = i / CX_STATE_BLOCK;
        const Vec4<float> m = m_value(__builtin_bit_cast(unsigned, load_up_to4(pm + i, k)), c.m_scale[block]);
        const Vec4<float> v = v_value(__builtin_bit_cast(unsigned, load_up_to4(pv + i, k)), c.v_scale[block]);
        store_up_to4(m_out + c.flat + i, from_float<E>(m), k);
        store_up_to4(v_out + c.flat + i, from_float<E>(v), k);
    }
}

__global__ __launch_bounds__(kBlock) void set_states_kernel(const Chunk* __restrict__ chunks,
                                                            const float* __restrict__ m_in,
                                                            const float* __restrict__ v_in) {
    const Chunk c = chunks[blockIdx.x];
    const int row = (threadIdx.x & 63) >> 4, r = threadIdx.x & 15;
    for (int q = (threadIdx.x >> 6) * kGroup; q < c.n; q += kBlock / 64 * kGroup) {
        const int at = q + row * CX_STATE_BLOCK, n = c.n - at, block = at / CX_STATE_BLOCK;
        Vec4<float> m[4], v[4];
        for (int j = 0; j < 4; ++j) {
            const int i = at + j * 64 + r * 4, k = c.n - i;
            m[j] = load_up_to4(m_in + c.flat + i, k);
            v[j] = load_up_to4(v_in + c.flat + i, k);
        }
        store_states<false>(m, v, static_cast<unsigned char*>(c.m) + at, static_cast<unsigned char*>(c.v) + at,
                            c.m_scale + block, c.v_scale + block, r, n);
    }
}

template <typename P, typename G, bool MASTER>
void launch_step(hipStream_t s, int bits, int n, const Chunk* chunks, int first, const GradArgs& g, const AdamwArgs& a) {
    if (bits == 32) adamw32_kernel<P, G, MASTER><<<n, kBlock, 0, s>>>(chunks, first, g, a);
    else adamw8_kernel<P, G, MASTER><<<n, kBlock, 0, s>>>(chunks, first, g, a);
}

template <typename P, bool MASTER>
void launch_step_for(int grad_type, hipStream_t s, int bits, int n, const Chunk* chunks, int first, const GradArgs& g,
                     const AdamwArgs& a) {
    if (grad_type == CX_F32) launch_step<P, float, MASTER>(s, bits, n, chunks, first, g, a);
    else if (grad_type == CX_BF16) launch_step<P, __bf16, MASTER>(s, bits, n, chunks, first, g, a);
    else launch_step<P, _Float16, MASTER>(s, bits, n, chunks, first, g, a);
}

}  // namespace

int launch_adamw(cx_handle h, cx_tensors t, const cx_grads* g, const cx_adamw_args* u) {
    AdamwArgs a = {};
    a.beta1 = (float)u->beta1;
    a.rest1 = (float)(1.0 - u->beta1);
    a.beta2 = (float)u->beta2;
    a.rest2 = (float)(1.0 - u->beta2);
    a.eps = (float)u->eps;
    a.scale = (float)u->scale;
    a.coefs = u->n_coefs ? u->d_coefs : nullptr;
    a.per_tensor = u->n_coefs != 1;
    a.skip = u->d_skip;
    if (u->d_step || u->d_lr) {
        AdamwRates* rates = reinterpret_cast<AdamwRates*>(t->d_rates);
        rates_kernel<<<1, 1, 0, h->stream>>>(u->d_step, u->step, u->d_lr, u->lr, u->beta1, u->beta2, u->weight_decay,
                                             u->d_skip, rates);
        CX_HIP(hipGetLastError());
        a.device_rates = rates;
    } else {
        a.rates = rates_of(u->lr, u->beta1, u->beta2, u->weight_decay, (double)u->step);
    }
    return for_grads(t, g, [&](int first, int n, const GradArgs& ga) -> int {
        const int bits = t->state_bits;
        if (t->param_type == CX_F32) launch_step_for<float, false>(g->type, h->stream, bits, n, t->d_chunks, first, ga, a);
        else if (t->param_type == CX_BF16 && t->masters) launch_step_for<__bf16, true>(g->type, h->stream, bits, n, t->d_chunks, first, ga, a);
        else if (t->param_type == CX_BF16) launch_step_for<__bf16, false>(g->type, h->stream, bits, n, t->d_chunks, first, ga, a);
        else if (t->masters) launch_step_for<_Float16, true>(g->type, h->stream, bits, n, t->d_chunks, first, ga, a);
        else launch_step_for<_Float16, false>(g->type, h->stream, bits, n, t->d_chunks, first, ga, a);
        CX_HIP(hipGetLastError());
        return CX_OK;
    });
}

int launch_adamw_states(cx_handle h, cx_tensors t, int dt, void* d_m, void* d_v) {
    if (t->chunks == 0) return CX_OK;
    if (dt == CX_F32) states_kernel<<<t->chunks, kBlock, 0, h->stream>>>(t->d_chunks, static_cast<float*>(d_m), static_cast<float*>(d_v));
    else if (dt == CX_BF16) states_kernel<<<t->chunks, kBlock, 0, h->stream>>>(t->d_chunks, static_cast<__bf16*>(d_m), static_cast<__bf16*>(d_v));
    else states_kernel<<<t->chunks, kBlock, 0, h->stream>>>(t->d_chunks, static_cast<_Float16*>(d_m), static_cast<_Float16*>(d_v));
    CX_HIP(hipGetLastError());
    return CX_OK;
}

int launch_adamw_set_states(cx_handle h, cx_tensors t, const float* d_m, const float* d_v) {
    if (t->chunks == 0) return CX_OK;
    set_states_kernel<<<t->chunks, kBlock, 0, h->stream>>>(t->d_chunks, d_m, d_v);
    CX_HIP(hipGetLastError());
    return CX_OK;
}

}  // namespace cx
