// The tensors of an optimizer step (cx_tensors): sizes, the pieces the kernels walk, and what the
// kernels over many tensors share.  Kernels: k_tensors.hip (norms, packing), k_adamw.hip.
#pragma once

#include "cx_common.hpp"

#include <type_traits>
#include <vector>

namespace cx {

enum { kFine = 0, kWide = 1, kCoarse = 2, kDivisions = 3 };

// One tensor.  A kernel reads one entry with scalar loads.
struct alignas(16) Tensor {
    long long n;          // elements
    long long flat;       // first element within the flat vector of all tensors
    int first[kDivisions];  // first piece in each of the divisions below
    int lead;             // its first fine piece is shorter by so many elements
    void* param;
    float* master;        // nullptr: none
    void* m;              // float or codes
    void* v;
    float* m_scale;       // 8-bit states only
    float* v_scale;
};

// The tensors are cut into pieces, one workgroup's work each; a tensor's last piece may be shorter.  `owner`
// says which tensor a piece belongs to (4 bytes a piece, and the tensors' table stays in the caches).
// kFine and kWide: what reads and writes, 4 or 8 elements a lane.  Pieces of one load per stream and lane: all
// workgroups in flight then walk through each buffer as one narrow front.  fp32 step on 25.6 M elements: 122 us
// with 1024 elements a piece, 128 with 2048, 141 with 4096, 151 with 16384 (loops over the piece), 159 with 65536.
// Where fp32 moments do not begin on a 128-byte line (tensors back to back), the first fine piece is shortened so
// that the others do: fp32 step on 64 Mi such elements 304 us, 332 us without.  (Packing, which reads what is
// aligned and writes what is not, or the other way round, gains nothing: 106 us without, 108 with, 100 M in bf16.)
// kCoarse: the sums of squares, which want few partial sums.
struct Pieces {
    const Tensor* tensors;
    const int* owner;
    int step;             // elements of a piece
    int first;            // first piece of the launch
};
struct Piece {
    Tensor t;
    int tensor;
    long long at;         // first element within the tensor
    int n;                // elements
};

// The launch's pieces, dealt out so that each of the 8 XCDs (workgroup b runs on XCD b mod 8) takes 32 in a
// row: fp32 step on 64 Mi elements 352 us dealt out one by one, 339 / 333 us with 4 / 16 in a row, 366 us with
// an eighth of the whole each.
constexpr int kXcds = 8, kRun = 32;
__device__ __forceinline__ int dealt(int b, int n) {
    constexpr int round = kXcds * kRun;
    return b < n / round * round ? b / round * round + b % kXcds * kRun + b % round / kXcds : b;
}

template <int WHICH> __device__ __forceinline__ Piece piece_of(const Pieces& ps) {
    Piece c;
    const int id = ps.first + dealt(blockIdx.x, gridDim.x);
    c.tensor = __builtin_amdgcn_readfirstlane(ps.owner[id]);
    c.t = ps.tensors[c.tensor];
    const long long from = (long long)(id - c.t.first[WHICH]) * ps.step - (WHICH == kFine ? c.t.lead : 0);
    c.at = max(from, 0ll);
    c.n = (int)(min(from + ps.step, c.t.n) - c.at);
    return c;
}

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

template <typename E, int N> using Vec = E __attribute__((ext_vector_type(N)));

// N elements at any address that is aligned to one: gfx950's vector loads and stores take it.  The addresses
// come out of a table, so the compiler has to be told that they are global memory.  Past the caches
// (nontemporal) unless `KEEP`: a step touches everything once (fp32 step, 64 Mi elements in pieces of 2048: 355 us,
// plain loads and stores 358 us, 25.6 M elements 128 and 147 us).
template <int N, bool KEEP = false, typename E>
__device__ __forceinline__ Vec<E, N> load(const E* p) {
    typedef Vec<E, N> V __attribute__((aligned(sizeof(E))));
    auto* g = (const __attribute__((address_space(1))) V*)p;
    if constexpr (KEEP) return *g;
    else return __builtin_nontemporal_load(g);
}
template <int N, typename E>
__device__ __forceinline__ void store(E* p, Vec<E, N> x) {
    typedef Vec<E, N> V __attribute__((aligned(sizeof(E))));
    __builtin_nontemporal_store(x, (__attribute__((address_space(1))) V*)p);
}
template <typename E> __device__ __forceinline__ __attribute__((address_space(1))) E* global(E* p) {
    return (__attribute__((address_space(1))) E*)p;
}
// The first `k` of them, zeros for the rest.  FULL: all of them, without asking.
template <int N, bool FULL = false, bool KEEP = false, typename E>
__device__ __forceinline__ Vec<E, N> load_some(const E* p, int k) {
    if (FULL || k >= N) return load<N, KEEP>(p);
    Vec<E, N> x = {};
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
        if (k > i) x[i] = global(p)[i];
    return x;
}
template <int N, bool FULL = false, typename E>
__device__ __forceinline__ void store_some(E* p, Vec<E, N> x, int k) {
    if (FULL || k >= N) return store<N>(p, x);
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
        if (k > i) global(p)[i] = x[i];
}
template <int N, typename E> __device__ __forceinline__ Vec<float, N> to_float(Vec<E, N> x) {
    return __builtin_convertvector(x, Vec<float, N>);
}
template <typename E, int N> __device__ __forceinline__ Vec<E, N> from_float(Vec<float, N> x) {
    return __builtin_convertvector(x, Vec<E, N>);  // to nearest, ties to even
}

// The gradient of a piece, nullptr where its tensor has none.
template <typename G> __device__ __forceinline__ const G* grad_of(const Piece& c, const GradArgs& g) {
    if (g.flat) return static_cast<const G*>(g.flat) + c.t.flat + c.at;
    const G* p = static_cast<const G*>(g.each[c.tensor - g.first]);
    return p ? p + c.at : nullptr;
}

// Calls body with true_type for a whole piece (no lane asks how many elements it has) and false_type for
// a tensor's last one.
template <int STEP, typename F> __device__ __forceinline__ void by_length(const Piece& c, F&& body) {
    if (c.n == STEP) body(std::true_type{});
    else body(std::false_type{});
}

// coef * scale of a piece's tensor
__device__ __forceinline__ float factor_of(const Piece& c, const float* coefs, int per_tensor, float scale) {
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
    long long total = 0;
    std::vector<long long> sizes, flat;     // per tensor; flat: its first element in the flat vector
    struct Division {
        int step = 0;                       // elements of a piece
        int pieces = 0;
        int longest = 0;                    // most pieces of one tensor
        std::vector<int> first;             // count + 1
        int* d_owner = nullptr;
        int* d_first = nullptr;             // `first` on the device
    } cut[cx::kDivisions];
    bool adamw = false;
    int param_type = 0, state_bits = 0;
    bool masters = false;
    // device
    void* memory = nullptr;                 // holds all of the following
    cx::Tensor* d_tensors = nullptr;
    double* d_partial = nullptr;            // per coarse piece: sum of the gradient's squares
    unsigned* d_done = nullptr;             // workgroups of small_norms_kernel that are through; 0 between launches
    float* d_rates = nullptr;               // what a device-side step count gives (AdamwRates)

    cx::Pieces pieces(int which, int from = 0) const {
        return {d_tensors, cut[which].d_owner, cut[which].step, from};
    }
};

namespace cx {

// Calls `launch(pieces, number of pieces, args)` for as many tensors at a time as one launch's arguments hold.
template <typename F> int for_grads(cx_tensors t, const cx_grads* g, int which, F&& launch) {
    const auto& cut = t->cut[which];
    GradArgs a;
    a.flat = g->flat;
    a.first = 0;
    if (cut.pieces == 0) return CX_OK;
    if (g->flat) return launch(t->pieces(which), cut.pieces, a);
    for (int first = 0; first < t->count; first += kGradsPerLaunch) {
        const int last = first + kGradsPerLaunch < t->count ? first + kGradsPerLaunch : t->count;
        a.first = first;
        for (int k = first; k < last; ++k) a.each[k - first] = g->each[k];
        const int from = cut.first[first], n = cut.first[last] - from;
        const int rc = n ? launch(t->pieces(which, from), n, a) : CX_OK;
        if (rc != CX_OK) return rc;
    }
    return CX_OK;
}

int launch_grad_norms(cx_handle h, cx_tensors t, const cx_grads* g, double scale, double max_norm, int each,
                      float* d_norms, float* d_coefs, int* d_nonfinite);
int launch_pack(cx_handle h, cx_tensors t, const cx_grads* g, const float* d_coefs, int n_coefs, float scale,
                const int* d_skip, float* out);
int launch_adamw(cx_handle h, cx_tensors t, const cx_grads* g, const cx_adamw_args* a, unsigned long long seed);
int launch_adamw_apply(cx_handle h, cx_tensors t, const float* d_moves, float scale, double lr, const float* d_lr,
                       double weight_decay);
int launch_adamw_states(cx_handle h, cx_tensors t, int dt, void* d_m, void* d_v);
int launch_adamw_set_states(cx_handle h, cx_tensors t, const float* d_m, const float* d_v);

}  // namespace cx
