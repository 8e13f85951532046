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

constexpr int kBlock = 256;   // 4 elements a lane: a piece of 1024

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
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float below = __builtin_fmaf(__builtin_sqrtf(v[k]), r.v_unit, a.eps);
        w[k] -= __builtin_fmaf(r.decay, w[k], r.step * (m[k] / below));
    }
    return w;
}

// One piece a workgroup, four elements a lane: everything is asked for before anything is used.
template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kBlock) void adamw32_kernel(Pieces ps, GradArgs ga, AdamwArgs a) {
    const Piece c = piece_of<kFine>(ps);
    const G* g = grad_of<G>(c, ga);
    if (!g || (a.skip && *a.skip)) return;
    const AdamwRates r = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    P* p = static_cast<P*>(c.t.param) + c.at;
    float *pm = static_cast<float*>(c.t.m) + c.at, *pv = static_cast<float*>(c.t.v) + c.at, *pw = c.t.master + c.at;
    const int i = threadIdx.x * 4, k = c.n - i;
    if (k <= 0) return;
    by_length(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const Vec4<G> gx = load_up_to4<FULL>(g + i, k);
        Vec4<float> m = load_up_to4<FULL>(pm + i, k), v = load_up_to4<FULL>(pv + i, k);
        Vec4<float> w;
        if constexpr (MASTER) w = load_up_to4<FULL>(pw + i, k);
        else w = to_float<P>(load_up_to4<FULL>(p + i, k));
        moments(to_float<G>(gx) * f, a, m, v);
        w = weights(w, m, v, a, r);
        store_up_to4<FULL>(pm + i, m, k);
        store_up_to4<FULL>(pv + i, v, k);
        if constexpr (MASTER) store_up_to4<FULL>(pw + i, w, k);
        store_up_to4<FULL>(p + i, from_float<P>(w), k);
    });
}

// ---- 8-bit moments ---------------------------------------------------------------------------
// A wave holds a block of 256 elements, four a lane.

constexpr float kTiny = 0x1p-100f;               // a block below is stored as zeros
constexpr float kVUnit = 0x1.ep-96f;             // V lies here before its bits are cut: exponent field 31, fraction 7/8
constexpr float kVBack = (float)(0x1p96 / 1.875);

// The wave's maximum, in every lane: four rotations within rows of 16 lanes, two broadcasts of a row's last
// lane to the rows behind it, then lane 63 has seen all.
__device__ __forceinline__ unsigned wave_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));  // row_bcast:15
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));  // row_bcast:31
    return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// The largest finite magnitude of the wave's values (floats of one sign are ordered like their bits).
__device__ __forceinline__ float block_max(Vec4<float> x) {
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned u = __float_as_uint(x[k]) & 0x7fffffffu;
        top = max(top, u < 0x7f800000u ? u : 0u);
    }
    return __uint_as_float(wave_max(top));
}

__device__ __forceinline__ Vec4<float> m_value(unsigned codes, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return Vec4<float>{lo[0], lo[1], hi[0], hi[1]} * scale;
}
__device__ __forceinline__ Vec4<float> v_value(unsigned codes, float scale) {
    Vec4<float> x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(((codes >> (8 * k)) & 255u) << 20);
    return x * kVBack * scale;
}
__device__ __forceinline__ unsigned m_codes(Vec4<float> m, float inverse) {
    m = m * inverse;
    const int u = __builtin_amdgcn_cvt_pk_fp8_f32(m[0], m[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[2], m[3], u, true);
}
// The value's own exponent and upper fraction bits, after a scaling that leaves 5 bits of exponent: small
// values run into the format's subnormals as they do into those of fp32.  Rounded to nearest.
__device__ __forceinline__ unsigned v_codes(Vec4<float> v, float inverse) {
    const Vec4<float> y = v * inverse * kVUnit;
    unsigned u = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned code = ((__float_as_uint(y[k]) + 0x80000u) >> 20) & 255u;   // (no finite value exceeds 255)
        u |= max(code, min(__float_as_uint(v[k]), 1u)) << (8 * k);                 // above 0: never 0
    }
    return u;
}

// Rounds the moments of the wave's block and stores them: this lane's four codes of each (k of them exist) and
// the block's scales.
template <bool FULL>
__device__ __forceinline__ void store_states(Vec4<float> m, Vec4<float> v, unsigned char* pm, unsigned char* pv, float* sm,
                                             float* sv, int k) {
    const float mt = block_max(m), vt = block_max(v);
    const bool m_kept = mt >= kTiny, v_kept = vt >= kTiny;
    const unsigned mc = m_codes(m, m_kept ? 448.0f / mt : 0.0f);
    const unsigned vc = v_kept ? v_codes(v, 1.0f / vt) : 0u;
    store_up_to4<FULL>(pm, __builtin_bit_cast(Vec4<unsigned char>, mc), k);
    store_up_to4<FULL>(pv, __builtin_bit_cast(Vec4<unsigned char>, vc), k);
    if ((threadIdx.x & 63) == 0) {
        *global(sm) = m_kept ? mt * (float)(1.0 / 448.0) : 0.0f;
        *global(sv) = v_kept ? vt : 0.0f;
    }
}

template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kBlock) void adamw8_kernel(Pieces ps, GradArgs ga, AdamwArgs a) {
    const Piece c = piece_of<kFine>(ps);
    const G* g = grad_of<G>(c, ga);
    if (!g || (a.skip && *a.skip)) return;
    const AdamwRates r = a.device_rates ? *a.device_rates : a.rates;
    const float f = factor_of(c, a.coefs, a.per_tensor, a.scale);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave * CX_STATE_BLOCK >= c.n) return;
    P* p = static_cast<P*>(c.t.param) + c.at;
    unsigned char *pm = static_cast<unsigned char*>(c.t.m) + c.at, *pv = static_cast<unsigned char*>(c.t.v) + c.at;
    float* pw = c.t.master + c.at;
    const long long block = c.at / CX_STATE_BLOCK + wave;
    float *sm = c.t.m_scale + block, *sv = c.t.v_scale + block;
    const int i = threadIdx.x * 4, k = c.n - i;
    by_length(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const Vec4<G> gx = load_up_to4<FULL>(g + i, k);
        const unsigned mc = __builtin_bit_cast(unsigned, load_up_to4<FULL>(pm + i, k));
        const unsigned vc = __builtin_bit_cast(unsigned, load_up_to4<FULL>(pv + i, k));
        Vec4<float> w;
        if constexpr (MASTER) w = load_up_to4<FULL>(pw + i, k);
        else w = to_float<P>(load_up_to4<FULL>(p + i, k));
        Vec4<float> m = m_value(mc, *global(sm)), v = v_value(vc, *global(sv));
        moments(to_float<G>(gx) * f, a, m, v);
        w = weights(w, m, v, a, r);
        if constexpr (MASTER) store_up_to4<FULL>(pw + i, w, k);
        store_up_to4<FULL>(p + i, from_float<P>(w), k);
        store_states<FULL>(m, v, pm + i, pv + i, sm, sv, k);
    });
}

template <typename E>
__global__ __launch_bounds__(kBlock) void states_kernel(Pieces ps, E* __restrict__ m_out, E* __restrict__ v_out) {
    const Piece c = piece_of<kFine>(ps);
    const unsigned char *pm = static_cast<const unsigned char*>(c.t.m) + c.at, *pv = static_cast<const unsigned char*>(c.t.v) + c.at;
    const int i = threadIdx.x * 4, k = c.n - i;
    if (k <= 0) return;
    const long long block = (c.at + i) / CX_STATE_BLOCK, to = c.t.flat + c.at + i;
    by_length(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        const unsigned mc = __builtin_bit_cast(unsigned, load_up_to4<FULL>(pm + i, k));
        const unsigned vc = __builtin_bit_cast(unsigned, load_up_to4<FULL>(pv + i, k));
        store_up_to4<FULL>(m_out + to, from_float<E>(m_value(mc, global(c.t.m_scale)[block])), k);
        store_up_to4<FULL>(v_out + to, from_float<E>(v_value(vc, global(c.t.v_scale)[block])), k);
    });
}

__global__ __launch_bounds__(kBlock) void set_states_kernel(Pieces ps, const float* __restrict__ m_in,
                                                            const float* __restrict__ v_in) {
    const Piece c = piece_of<kFine>(ps);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave * CX_STATE_BLOCK >= c.n) return;
    const int i = threadIdx.x * 4, k = c.n - i;
    const long long from = c.t.flat + c.at + i, block = c.at / CX_STATE_BLOCK + wave;
    store_states<false>(load_up_to4(m_in + from, k), load_up_to4(v_in + from, k), static_cast<unsigned char*>(c.t.m) + c.at + i,
                 static_cast<unsigned char*>(c.t.v) + c.at + i, c.t.m_scale + block, c.t.v_scale + block, k);
}

template <typename P, typename G, bool MASTER>
void launch_step(hipStream_t s, int bits, int n, const Pieces& ps, const GradArgs& g, const AdamwArgs& a) {
    if (bits == 32) adamw32_kernel<P, G, MASTER><<<n, kBlock, 0, s>>>(ps, g, a);
    else adamw8_kernel<P, G, MASTER><<<n, kBlock, 0, s>>>(ps, g, a);
}

template <typename P, bool MASTER>
void launch_step_for(int grad_type, hipStream_t s, int bits, int n, const Pieces& ps, const GradArgs& g, const AdamwArgs& a) {
    if (grad_type == CX_F32) launch_step<P, float, MASTER>(s, bits, n, ps, g, a);
    else if (grad_type == CX_BF16) launch_step<P, __bf16, MASTER>(s, bits, n, ps, g, a);
    else launch_step<P, _Float16, MASTER>(s, bits, n, ps, g, a);
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
    return for_grads(t, g, kFine, [&](const Pieces& ps, int n, const GradArgs& ga) -> int {
        const int bits = t->state_bits;
        if (t->param_type == CX_F32) launch_step_for<float, false>(g->type, h->stream, bits, n, ps, ga, a);
        else if (t->param_type == CX_BF16 && t->masters) launch_step_for<__bf16, true>(g->type, h->stream, bits, n, ps, ga, a);
        else if (t->param_type == CX_BF16) launch_step_for<__bf16, false>(g->type, h->stream, bits, n, ps, ga, a);
        else if (t->masters) launch_step_for<_Float16, true>(g->type, h->stream, bits, n, ps, ga, a);
        else launch_step_for<_Float16, false>(g->type, h->stream, bits, n, ps, ga, a);
        CX_HIP(hipGetLastError());
        return CX_OK;
    });
}

int launch_adamw_states(cx_handle h, cx_tensors t, int dt, void* d_m, void* d_v) {
    const int n = t->cut[kFine].pieces;
    if (n == 0) return CX_OK;
    const Pieces ps = t->pieces(kFine);
    if (dt == CX_F32) states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<float*>(d_m), static_cast<float*>(d_v));
    else if (dt == CX_BF16) states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<__bf16*>(d_m), static_cast<__bf16*>(d_v));
    else states_kernel<<<n, kBlock, 0, h->stream>>>(ps, static_cast<_Float16*>(d_m), static_cast<_Float16*>(d_v));
    CX_HIP(hipGetLastError());
    return CX_OK;
}

int launch_adamw_set_states(cx_handle h, cx_tensors t, const float* d_m, const float* d_v) {
    const int n = t->cut[kFine].pieces;
    if (n == 0) return CX_OK;
    set_states_kernel<<<n, kBlock, 0, h->stream>>>(t->pieces(kFine), d_m, d_v);
    CX_HIP(hipGetLastError());
    return CX_OK;
}

}  // namespace cx
