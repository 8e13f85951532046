// The tensors of an optimizer step (cx_tensors): sizes, the pieces the kernels walk, and what the
// kernels over many tensors share.  Kernels: k_tensors.hip (norms, packing), k_adamw.hip.
#pragma once

#include "cx_common.hpp"

#include <vector>

namespace cx {

// One workgroup's piece of one tensor.  The addresses are those of the piece's first element; a kernel
// reads one Chunk with scalar loads and needs no other table.
struct alignas(16) Chunk {
    long long at;      // first element within its tensor
    long long flat;    // first element within the flat vector of all tensors
    int tensor;
    int n;             // elements
    void* param;
    float* master;     // nullptr: none
    void* m;           // float or codes
    void* v;
    float* m_scale;    // 8-bit states only: the scale of the piece's first block
    float* v_scale;
};

// A launch's gradients: one flat vector, or the addresses of up to kGradsPerLaunch tensors.  They travel as
// kernel arguments, because gradients move between steps where parameters stay: no upload to wait for or to
// keep alive, and a captured graph holds them.
constexpr int kGradsPerLaunch = 448;
struct GradArgs {
    const void* flat;
    int first;         // tensor that each[0] belongs to
    const void* each[kGradsPerLaunch];
};

template <int DT> struct Num;
template <> struct Num<CX_F32> { using type = float; };
template <> struct Num<CX_BF16> { using type = __bf16; };
template <> struct Num<CX_F16> { using type = _Float16; };

template <typename E> using Vec4 = E __attribute__((ext_vector_type(4)));

// Four elements at any address that is aligned to one: gfx950's vector loads and stores take it.
template <typename E>
__device__ __forceinline__ Vec4<E> load4(const E* p) {
    typedef Vec4<E> V __attribute__((aligned(sizeof(E))));
    return *reinterpret_cast<const V*>(p);
}
template <typename E>
__device__ __forceinline__ void store4(E* p, Vec4<E> x) {
    typedef Vec4<E> V __attribute__((aligned(sizeof(E))));
    *reinterpret_cast<V*>(p) = x;
}
// The first `k` (1..4) of them, zeros for the rest.
template <typename E>
__device__ __forceinline__ Vec4<E> load_up_to4(const E* p, int k) {
    if (k >= 4) return load4(p);
    Vec4<E> x = {};
    if (k > 0) x[0] = p[0];
    if (k > 1) x[1] = p[1];
    if (k > 2) x[2] = p[2];
    return x;
}
template <typename E>
__device__ __forceinline__ void store_up_to4(E* p, Vec4<E> x, int k) {
    if (k >= 4) return store4(p, x);
    if (k > 0) p[0] = x[0];
    if (k > 1) p[1] = x[1];
    if (k > 2) p[2] = x[2];
}
template <typename E> __device__ __forceinline__ Vec4<float> to_float(Vec4<E> x) {
    return __builtin_convertvector(x, Vec4<float>);
}
template <typename E> __device__ __forceinline__ Vec4<E> from_float(Vec4<float> x) {
    return __builtin_convertvector(x, Vec4<E>);  // to nearest, ties to even
}

// The gradient of a piece, nullptr where its tensor has none.
template <typename G> __device__ __forceinline__ const G* grad_of(const Chunk& c, const GradArgs& g) {
    if (g.flat) return static_cast<const G*>(g.flat) + c.flat;
    const G* p = static_cast<const G*>(g.each[c.tensor - g.first]);
    return p ? p + c.at : nullptr;
}

// coef * scale of a piece's tensor
__device__ __forceinline__ float factor_of(const Chunk& c, const float* coefs, int per_tensor, float scale) {
    return coefs ? coefs[per_tensor ? c.tensor : 0] * scale : scale;
}

// Runs on the set's device whatever the caller's current one is.
struct DeviceScope {
    int before = -1;
    hipError_t error = hipSuccess;
    explicit DeviceScope(int device) {
        int now = 0;
        error = hipGetDevice(&now);
        if (error == hipSuccess && now != device) {
            error = hipSetDevice(device);
            if (error == hipSuccess) before = now;
        }
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

}  // namespace cx

struct cx_tensors_s {
    int device = 0;
    int count = 0;
    int chunks = 0;
    long long total = 0;
    std::vector<long long> sizes, flat;     // per tensor; flat: its first element in the flat vector
    std::vector<int> first_chunk;           // count + 1
    bool adamw = false;
    int param_type = 0, state_bits = 0;
    bool masters = false;
    // device
    cx::Chunk* d_chunks = nullptr;
    int* d_first_chunk = nullptr;           // count + 1
    double* d_partial = nullptr;            // per piece: sum of the gradient's squares
    float* d_rates = nullptr;               // what a device-side step count gives (AdamwRates)
};

namespace cx {

// Calls `launch(first_chunk, n_chunks, args)` for as many tensors at a time as one launch's arguments hold.
template <typename F> int for_grads(cx_tensors t, const cx_grads* g, F&& launch) {
    GradArgs a;
    a.flat = g->flat;
    a.first = 0;
    if (t->chunks == 0) return CX_OK;
    if (g->flat) return launch(0, t->chunks, a);
    for (int first = 0; first < t->count; first += kGradsPerLaunch) {
        const int last = first + kGradsPerLaunch < t->count ? first + kGradsPerLaunch : t->count;
        a.first = first;
        for (int k = first; k < last; ++k) a.each[k - first] = g->each[k];
        const int from = t->first_chunk[first], n = t->first_chunk[last] - from;
        const int rc = n ? launch(from, n, a) : CX_OK;
        if (rc != CX_OK) return rc;
    }
    return CX_OK;
}

int launch_grad_norms(cx_handle h, cx_tensors t, const cx_grads* g, double scale, double max_norm, int each,
                      float* d_norms, float* d_coefs, int* d_nonfinite);
int launch_pack(cx_handle h, cx_tensors t, const cx_grads* g, const float* d_coefs, int n_coefs, float scale,
                const int* d_skip, float* out);
int launch_adamw(cx_handle h, cx_tensors t, const cx_grads* g, const cx_adamw_args* a);
int launch_adamw_states(cx_handle h, cx_tensors t, int dt, void* d_m, void* d_v);
int launch_adamw_set_states(cx_handle h, cx_tensors t, const float* d_m, const float* d_v);

}  // namespace cx
