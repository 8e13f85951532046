// Many tensors at once: the set itself (cx_tensors_*), the gradients' norms and clip coefficients, and
// the flat vector that the compressor takes (keras/comprex_optimizer.py:97-133 of the reference does the
// latter two tensor after tensor).
#include "cx_tensors.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <memory>

namespace cx {

namespace {

constexpr int kBlock = 256;

__device__ __forceinline__ double wave_sum(double x) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// The block's sum, in thread 0.
template <int BLOCK> __device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[BLOCK / 64];
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int k = 0; k < BLOCK / 64; ++k) s += part[k];
    return s;
}

template <int N> __device__ __forceinline__ double add_squares(double s, Vec<float, N> x) {
#pragma unroll
    for (int k = 0; k < N; ++k) s = __builtin_fma((double)x[k], (double)x[k], s);
    return s;
}

// The piece's sum of g^2, in thread 0.  64 bits: the squares of finite floats do not overflow there.
template <typename G> __device__ __forceinline__ double piece_squares(const Piece& c, const G* g) {
    double s = 0.0;
    if (g) {
        constexpr int N = 16 / sizeof(G);  // 16 bytes a load, four of them asked for at a time
        int i = threadIdx.x * N;
        for (; i + 3 * kBlock * N + N <= c.n; i += kBlock * N * 4) {
            Vec<G, N> x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = load<N, true>(g + i + j * kBlock * N);
#pragma unroll
            for (int j = 0; j < 4; ++j) s = add_squares<N>(s, to_float<N>(x[j]));
        }
        for (; i < c.n; i += kBlock * N) s = add_squares<N>(s, to_float<N>(load_some<N, false, true>(g + i, c.n - i)));
    }
    return block_sum<kBlock>(s);
}

// What becomes of the sums: entry t < count is tensor t, entry `count` all of them.
struct NormsOut {
    int count;
    double scale, max_norm;
    int each;
    float *norms, *coefs;
    int* nonfinite;

    __device__ __forceinline__ void put(int t, double s) const {
        const double norm = sqrt(s) * scale;
        if (norms) norms[t] = (float)norm;
        const float coef = norm > max_norm ? (float)(max_norm / norm) : 1.0f;
        if (coefs && each && t < count) coefs[t] = coef;
        if (coefs && !each && t == count) coefs[0] = coef;
        if (nonfinite && t == count) *nonfinite = s <= 1.7976931348623157e308 ? 0 : 1;
    }
};

template <typename G>
__global__ __launch_bounds__(kBlock) void squares_kernel(Pieces ps, GradArgs ga, double* __restrict__ partial) {
    const Piece c = piece_of<kCoarse>(ps);
    const double s = piece_squares(c, grad_of<G>(c, ga));
    if (threadIdx.x == 0) partial[ps.first + dealt(blockIdx.x, gridDim.x)] = s;
}

// Block t < count: tensor t's norm; block `count`: that of all, from all pieces' sums in a fixed order.
constexpr int kNormsBlock = 1024;
__global__ __launch_bounds__(kNormsBlock) void norms_kernel(const double* __restrict__ partial,
                                                       const int* __restrict__ first_piece, NormsOut out) {
    const int t = blockIdx.x;
    const int from = t < out.count ? first_piece[t] : 0, to = first_piece[t < out.count ? t + 1 : out.count];
    double s = 0.0;
    int i = from + threadIdx.x;
    for (; i + 3 * kNormsBlock < to; i += 4 * kNormsBlock) {  // loads of one turn together
        const double a = partial[i], b = partial[i + kNormsBlock], c = partial[i + 2 * kNormsBlock], d = partial[i + 3 * kNormsBlock];
        s += (a + b) + (c + d);
    }
    for (; i < to; i += kNormsBlock) s += partial[i];
    s = block_sum<kNormsBlock>(s);
    if (threadIdx.x == 0) out.put(t, s);
}

// Both in one launch, for sets of at most kBlock pieces and fewer tensors, the longest of kSmallTensor pieces: the
// workgroup that finishes last (`done` counts them, and is 0 again behind the launch) makes the norms.  No workgroup
// waits.  One launch against two, us a call: 61 706 elements in 10 tensors 5.9 and 9.1, 2^18 in 50 (100 pieces) 6.3 and
// 9.1, 638 976 in 200 (200 pieces) 8.6 and 9.4, 2^18 in one (64 pieces, which one thread adds) 7.6 and 9.1; beyond the
// limits 2^20 in one tensor 17.7 and 9.0.
constexpr int kSmallTensor = 64;
template <typename G>
__global__ __launch_bounds__(kBlock) void small_norms_kernel(Pieces ps, GradArgs ga, double* partial, unsigned* done,
                                                             const int* __restrict__ first_piece, NormsOut out) {
    __shared__ double sums[kBlock];
    __shared__ unsigned last;
    const Piece c = piece_of<kCoarse>(ps);
    const double mine = piece_squares(c, grad_of<G>(c, ga));
    if (threadIdx.x == 0) {
        __hip_atomic_store(partial + dealt(blockIdx.x, gridDim.x), mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    const int pieces = gridDim.x, i = threadIdx.x;
    const double x = i < pieces ? __hip_atomic_load(partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    sums[i] = x;
    if (i == 0) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double all = block_sum<kBlock>(x);  // (its barrier is the one that `sums` needs)
    if (i < out.count) {
        double s = 0.0;
        for (int k = first_piece[i]; k < first_piece[i + 1]; ++k) s += sums[k];
        out.put(i, s);
    }
    if (i == out.count) out.put(i, all);
}

template <typename G>
__global__ __launch_bounds__(kBlock) void pack_kernel(Pieces ps, GradArgs ga, const float* __restrict__ coefs, int per_tensor, float scale,
                                                      const int* __restrict__ skip, float* out) {
    const Piece c = piece_of<kFine>(ps);
    const G* g = grad_of<G>(c, ga);
    float* to = out + c.t.flat + c.at;
    const bool zeros = !g || (skip && *skip);
    const float f = factor_of(c, coefs, per_tensor, scale);
    const int i = threadIdx.x * 4, k = c.n - i;
    if (k <= 0) return;
    by_length<kBlock * 4>(c, [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        if (zeros) store_some<4, FULL>(to + i, Vec<float, 4>{}, k);
        else store_some<4, FULL>(to + i, to_float<4>(load_some<4, FULL>(g + i, k)) * f, k);
    });
}

// Elements of a coarse piece: few enough partial sums, enough workgroups.  Sums and norms of 25.6 M fp32 gradients:
// 23.4 us with 4096, 22.3 with 8192, 22.4 with 16384; of 100 M in bf16 48, 43 and 43.5 us.
int coarse_step(long long total) {
    long long c = total > (1ll << 24) ? 8192 : 4096;
    while (c < 65536 && c * 16384 < total) c *= 2;
    return (int)c;
}

// A launch has fewer than 2^32 threads, 256 for each piece of 1024 elements.
constexpr long long kMostElements = 1ll << 33;
constexpr int kMostTensors = 1 << 20;

constexpr int kLine = 32;  // fp32 elements of 128 bytes

struct Span {
    uintptr_t from, to;
};

void add_span(std::vector<Span>& spans, const void* p, long long bytes) {
    if (p && bytes > 0) spans.push_back({reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + (uintptr_t)bytes});
}

int element_bytes(int dt) { return dt == CX_F32 ? 4 : 2; }

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

}  // namespace

static_assert(kBlock <= kGradsPerLaunch, "the gradients of a small set fit one launch");

#define CX_NUM_DISPATCH(dt, CALL)                                                     \
    switch (dt) {                                                                     \
        case CX_F32: { using G = Num<CX_F32>::type; CALL; } break;                    \
        case CX_BF16: { using G = Num<CX_BF16>::type; CALL; } break;                  \
        default: { using G = Num<CX_F16>::type; CALL; } break;                        \
    }

int launch_grad_norms(cx_handle h, cx_tensors t, const cx_grads* g, double scale, double max_norm, int each,
                      float* d_norms, float* d_coefs, int* d_nonfinite) {
    const NormsOut out = {t->count, std::fabs(scale), max_norm, each, d_norms, d_coefs, d_nonfinite};
    const auto& cut = t->cut[kCoarse];
    const bool small = cut.pieces > 0 && cut.pieces <= kBlock && t->count < kBlock &&  // (one launch's gradients)
                       cut.longest <= kSmallTensor;
    int rc = for_grads(t, g, kCoarse, [&](const Pieces& ps, int n, const GradArgs& a) -> int {
        if (small)
            CX_NUM_DISPATCH(g->type, (small_norms_kernel<G><<<n, kBlock, 0, h->stream>>>(ps, a, t->d_partial, t->d_done,
                                                                                         cut.d_first, out)))
        else
            CX_NUM_DISPATCH(g->type, (squares_kernel<G><<<n, kBlock, 0, h->stream>>>(ps, a, t->d_partial)))
        CX_HIP(hipGetLastError());
        return CX_OK;
    });
    if (rc != CX_OK || small) return rc;
    norms_kernel<<<t->count + 1, kNormsBlock, 0, h->stream>>>(t->d_partial, cut.d_first, out);
    CX_HIP(hipGetLastError());
    return CX_OK;
}

int launch_pack(cx_handle h, cx_tensors t, const cx_grads* g, const float* d_coefs, int n_coefs, float scale,
                const int* d_skip, float* out) {
    return for_grads(t, g, kFine, [&](const Pieces& ps, int n, const GradArgs& a) -> int {
        CX_NUM_DISPATCH(g->type, (pack_kernel<G><<<n, kBlock, 0, h->stream>>>(ps, a, d_coefs,
                                                                              n_coefs != 1, scale, d_skip, out)));
        CX_HIP(hipGetLastError());
        return CX_OK;
    });
}

}  // namespace cx

using namespace cx;

namespace {

bool number_type(int dt) { return dt == CX_F32 || dt == CX_BF16 || dt == CX_F16; }

// What every call over a set checks first.
int check_set(cx_handle h, cx_tensors t, const char* who) {
    if (!h || !t) return fail(CX_ERR_INVALID, "%s: null handle or set", who);
    if (h->device != t->device)
        return fail(CX_ERR_INVALID, "%s: the set lives on device %d, the handle on %d", who, t->device, h->device);
    return CX_OK;
}

int check_grads(cx_tensors t, const cx_grads* g, const char* who) {
    if (!g || !number_type(g->type)) return fail(CX_ERR_INVALID, "%s: gradients are fp32, bf16 or fp16", who);
    if (t->total > 0 && !g->each == !g->flat)
        return fail(CX_ERR_INVALID, "%s: needs either the tensors' gradients or the flat vector", who);
    const int bytes = element_bytes(g->type);
    if (g->flat && !aligned_to(g->flat, bytes)) return fail(CX_ERR_INVALID, "%s: misaligned gradient", who);
    if (g->each)
        for (int k = 0; k < t->count; ++k)
            if (!aligned_to(g->each[k], bytes)) return fail(CX_ERR_INVALID, "%s: misaligned gradient %d", who, k);
    return CX_OK;
}

// A flat output lies apart from the gradients, or an element on the gradient it is made of.
int check_apart(cx_tensors t, const cx_grads* grads, const float* out, const char* who) {
    const char *lo = reinterpret_cast<const char*>(out), *hi = lo + t->total * 4;
    const int bytes = element_bytes(grads->type);
    for (int k = 0; k < t->count; ++k) {
        if (t->sizes[k] == 0) continue;  // (of an empty set neither form of the gradients need be there)
        const char* g = grads->flat ? static_cast<const char*>(grads->flat) + t->flat[k] * bytes
                                    : static_cast<const char*>(grads->each[k]);
        if (!g || g >= hi || g + t->sizes[k] * bytes <= lo) continue;
        if (grads->type != CX_F32 || g != lo + t->flat[k] * 4)
            return fail(CX_ERR_INVALID, "%s: the output overlaps gradient %d", who, k);
    }
    return CX_OK;
}

int check_coefs(cx_tensors t, const float* d_coefs, int n_coefs, const char* who) {
    if (n_coefs != 0 && n_coefs != 1 && n_coefs != t->count)
        return fail(CX_ERR_SIZE_MISMATCH, "%s: %d coefficients for %d tensors", who, n_coefs, t->count);
    if (n_coefs != 0 && !d_coefs) return fail(CX_ERR_INVALID, "%s: null coefficients", who);
    return CX_OK;
}

}  // namespace

static int create_tensors(cx_tensors* out, cx_handle h, int count, const long long* sizes, const cx_adamw_state* state) {
    if (!out) return fail(CX_ERR_INVALID, "cx_tensors_create: null output");
    *out = nullptr;
    if (!h || count < 0 || count > kMostTensors || (count > 0 && !sizes)) return fail(CX_ERR_INVALID, "cx_tensors_create: bad arguments");
    long long total = 0;
    for (int k = 0; k < count; ++k) {
        if (sizes[k] < 0) return fail(CX_ERR_INVALID, "cx_tensors_create: tensor %d has a size of %lld", k, sizes[k]);
        if (sizes[k] > kMostElements || (total += sizes[k]) > kMostElements)
            return fail(CX_ERR_INVALID, "cx_tensors_create: more than %lld elements: make more sets", kMostElements);
    }
    if (state) {
        if (!number_type(state->param_type))
            return fail(CX_ERR_INVALID, "cx_tensors_create: parameters are fp32, bf16 or fp16");
        if (state->state_bits != 32 && state->state_bits != 8)
            return fail(CX_ERR_INVALID, "cx_tensors_create: states have 32 or 8 bits, not %d", state->state_bits);
        if (state->masters && state->param_type == CX_F32)
            return fail(CX_ERR_INVALID, "cx_tensors_create: fp32 parameters have no masters");
        const bool small = state->state_bits == 8;
        if (count > 0 && (!state->params || !state->exp_avg || !state->exp_avg_sq ||
                          small != (state->exp_avg_scales != nullptr) || small != (state->exp_avg_sq_scales != nullptr)))
            return fail(CX_ERR_INVALID, "cx_tensors_create: a list of the state is missing or superfluous");
        std::vector<Span> spans;
        for (int k = 0; k < count; ++k) {
            const long long n = sizes[k], blocks = (n + CX_STATE_BLOCK - 1) / CX_STATE_BLOCK;
            if (n == 0) continue;
            const int pb = element_bytes(state->param_type), sb = small ? 1 : 4;
            if (!state->params[k] || !state->exp_avg[k] || !state->exp_avg_sq[k] ||
                (state->masters && !state->masters[k]) ||
                (small && (!state->exp_avg_scales[k] || !state->exp_avg_sq_scales[k])))
                return fail(CX_ERR_INVALID, "cx_tensors_create: tensor %d has a null buffer", k);
            if (!aligned_to(state->params[k], pb) || !aligned_to(state->exp_avg[k], sb) ||
                !aligned_to(state->exp_avg_sq[k], sb) || (state->masters && !aligned_to(state->masters[k], 4)) ||
                (small && (!aligned_to(state->exp_avg_scales[k], 4) || !aligned_to(state->exp_avg_sq_scales[k], 4))))
                return fail(CX_ERR_INVALID, "cx_tensors_create: tensor %d has a misaligned buffer", k);
            add_span(spans, state->params[k], n * pb);
            add_span(spans, state->exp_avg[k], n * sb);
            add_span(spans, state->exp_avg_sq[k], n * sb);
            if (state->masters) add_span(spans, state->masters[k], n * 4);
            if (small) {
                add_span(spans, state->exp_avg_scales[k], blocks * 4);
                add_span(spans, state->exp_avg_sq_scales[k], blocks * 4);
            }
        }
        std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].from < spans[i - 1].to)
                return fail(CX_ERR_INVALID, "cx_tensors_create: two of the buffers overlap (a tensor given twice?)");
    }

    DeviceScope on(h->device);
    CX_HIP(on.error);
    std::unique_ptr<cx_tensors_s, int (*)(cx_tensors)> made(new cx_tensors_s(), cx_tensors_destroy);
    cx_tensors t = made.get();
    t->device = h->device;
    t->count = count;
    t->total = total;
    t->adamw = state != nullptr;
    if (state) {
        t->param_type = state->param_type;
        t->state_bits = state->state_bits;
        t->masters = state->masters != nullptr;
    }
    t->cut[kFine].step = kBlock * 4;
    t->cut[kWide].step = kBlock * 8;
    t->cut[kCoarse].step = coarse_step(total);
    std::vector<Tensor> tensors(count);
    std::vector<int> owner[kDivisions];
    long long flat = 0;
    for (int k = 0; k < count; ++k) {
        Tensor& x = tensors[k];
        x = Tensor{};
        x.n = sizes[k];
        x.flat = flat;
        if (state && sizes[k] > 0) {
            x.param = state->params[k];
            x.master = state->masters ? state->masters[k] : nullptr;
            x.m = state->exp_avg[k];
            x.v = state->exp_avg_sq[k];
            if (state->state_bits == 8) {
                x.m_scale = state->exp_avg_scales[k];
                x.v_scale = state->exp_avg_sq_scales[k];
            }
        }
        if (state && state->state_bits == 32) x.lead = (int)(reinterpret_cast<uintptr_t>(x.m) / 4 % kLine);
        for (int w = 0; w < kDivisions; ++w) {
            x.first[w] = (int)owner[w].size();
            t->cut[w].first.push_back(x.first[w]);
            const long long n = sizes[k] > 0 && w == kFine ? sizes[k] + x.lead : sizes[k];
            const int pieces = (int)((n + t->cut[w].step - 1) / t->cut[w].step);
            owner[w].insert(owner[w].end(), pieces, k);
            t->cut[w].longest = std::max(t->cut[w].longest, pieces);
        }
        t->sizes.push_back(sizes[k]);
        t->flat.push_back(flat);
        flat += sizes[k];
    }
    // one allocation: the tables, uploaded at once, and the scratch behind them
    std::vector<char> tables;
    size_t bytes = 0;
    auto place = [&](const void* from, size_t n) {  // where it will lie
        const size_t at = bytes;
        bytes = at + (n + 255) / 256 * 256;
        if (from) {
            tables.resize(bytes);
            if (n) std::memcpy(tables.data() + at, from, n);
        }
        return at;
    };
    const size_t at_tensors = place(tensors.data(), tensors.size() * sizeof(Tensor));
    size_t at_owner[kDivisions], at_first[kDivisions];
    for (int w = 0; w < kDivisions; ++w) {
        auto& cut = t->cut[w];
        cut.pieces = (int)owner[w].size();
        cut.first.push_back(cut.pieces);
        at_owner[w] = place(owner[w].data(), owner[w].size() * sizeof(int));
        at_first[w] = place(cut.first.data(), cut.first.size() * sizeof(int));
    }
    const unsigned zero = 0;
    const size_t at_done = place(&zero, sizeof zero);
    const size_t at_rates = place(nullptr, 256);
    const size_t at_partial = place(nullptr, t->cut[kCoarse].pieces * sizeof(double));
    hipError_t e = hipMalloc(&t->memory, bytes);
    if (e == hipSuccess) e = hipMemcpyAsync(t->memory, tables.data(), tables.size(), hipMemcpyHostToDevice, h->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->stream);  // the host's tables go away
    if (e != hipSuccess) return fail(CX_ERR_HIP, "cx_tensors_create: %s", hipGetErrorString(e));
    char* base = static_cast<char*>(t->memory);
    t->d_tensors = reinterpret_cast<Tensor*>(base + at_tensors);
    for (int w = 0; w < kDivisions; ++w) {
        t->cut[w].d_owner = reinterpret_cast<int*>(base + at_owner[w]);
        t->cut[w].d_first = reinterpret_cast<int*>(base + at_first[w]);
    }
    t->d_done = reinterpret_cast<unsigned*>(base + at_done);
    t->d_rates = reinterpret_cast<float*>(base + at_rates);
    t->d_partial = reinterpret_cast<double*>(base + at_partial);
    *out = made.release();
    return CX_OK;
}

extern "C" {

int cx_tensors_create(cx_tensors* out, cx_handle h, int count, const long long* sizes, const cx_adamw_state* state) {
    try {
        return create_tensors(out, h, count, sizes, state);
    } catch (const std::exception& e) {  // the host tables did not fit
        return fail(CX_ERR_INVALID, "cx_tensors_create: %s", e.what());
    }
}

int cx_tensors_destroy(cx_tensors t) {
    if (!t) return CX_OK;
    DeviceScope on(t->device);
    if (t->memory) (void)hipFree(t->memory);  // waits for the device
    delete t;
    return CX_OK;
}

int cx_grad_norms(cx_handle h, cx_tensors t, const cx_grads* grads, double scale, double max_norm, int each,
                  float* d_norms, float* d_coefs, int* d_nonfinite) {
    int rc = check_set(h, t, "cx_grad_norms");
    if (rc == CX_OK) rc = check_grads(t, grads, "cx_grad_norms");
    if (rc != CX_OK) return rc;
    if (!(max_norm > 0.0)) return fail(CX_ERR_INVALID, "cx_grad_norms: max_norm must be above 0");
    if (!std::isfinite(scale)) return fail(CX_ERR_INVALID, "cx_grad_norms: scale must be finite");
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_grad_norms(h, t, grads, scale, max_norm, each != 0, d_norms, d_coefs, d_nonfinite);
}

int cx_pack(cx_handle h, cx_tensors t, const cx_grads* grads, const float* d_coefs, int n_coefs, double scale,
            const int* d_skip, float* out) {
    int rc = check_set(h, t, "cx_pack");
    if (rc == CX_OK) rc = check_grads(t, grads, "cx_pack");
    if (rc == CX_OK) rc = check_coefs(t, d_coefs, n_coefs, "cx_pack");
    if (rc != CX_OK) return rc;
    if (!std::isfinite((float)scale)) return fail(CX_ERR_INVALID, "cx_pack: scale must be finite in fp32");
    if ((!out && t->total > 0) || !aligned_to(out, 4)) return fail(CX_ERR_INVALID, "cx_pack: null or misaligned output");
    rc = check_apart(t, grads, out, "cx_pack");
    if (rc != CX_OK) return rc;
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_pack(h, t, grads, n_coefs ? d_coefs : nullptr, n_coefs, (float)scale, d_skip, out);
}

int cx_adamw_step(cx_handle h, cx_tensors t, const cx_grads* grads, const cx_adamw_args* a) {
    return cx_adamw_step_seeded(h, t, grads, a, 0);
}

int cx_adamw_step_seeded(cx_handle h, cx_tensors t, const cx_grads* grads, const cx_adamw_args* a, unsigned long long seed) {
    int rc = check_set(h, t, "cx_adamw_step");
    if (rc == CX_OK) rc = check_grads(t, grads, "cx_adamw_step");
    if (rc == CX_OK && !a) rc = fail(CX_ERR_INVALID, "cx_adamw_step: null arguments");
    if (rc == CX_OK) rc = check_coefs(t, a->d_coefs, a->n_coefs, "cx_adamw_step");
    if (rc != CX_OK) return rc;
    if (!t->adamw) return fail(CX_ERR_INVALID, "cx_adamw_step: the set was made without a state");
    if (!a->d_lr && !(a->lr >= 0.0 && std::isfinite((float)a->lr)))
        return fail(CX_ERR_INVALID, "cx_adamw_step: the learning rate must be finite and not negative");
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0))
        return fail(CX_ERR_INVALID, "cx_adamw_step: the betas must lie in [0, 1)");
    if (!((float)a->eps >= 1e-20f && std::isfinite((float)a->eps)))
        return fail(CX_ERR_INVALID, "cx_adamw_step: eps must be finite and at least 1e-20");
    if (!(a->weight_decay >= 0.0 && std::isfinite((float)a->weight_decay)))
        return fail(CX_ERR_INVALID, "cx_adamw_step: the weight decay must be finite and not negative");
    if (!std::isfinite((float)a->scale)) return fail(CX_ERR_INVALID, "cx_adamw_step: scale must be finite");
    if (!aligned_to(a->d_moves, 4)) return fail(CX_ERR_INVALID, "cx_adamw_step: misaligned moves");
    if (a->d_moves && (rc = check_apart(t, grads, a->d_moves, "cx_adamw_step")) != CX_OK) return rc;
    if (!a->d_step && a->step < 1) return fail(CX_ERR_INVALID, "cx_adamw_step: steps count from 1");
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_adamw(h, t, grads, a, seed);
}

int cx_adamw_apply(cx_handle h, cx_tensors t, const float* d_moves, double scale, double lr, const float* d_lr,
                   double weight_decay) {
    const int rc = check_set(h, t, "cx_adamw_apply");
    if (rc != CX_OK) return rc;
    if (!t->adamw) return fail(CX_ERR_INVALID, "cx_adamw_apply: the set was made without a state");
    if ((!d_moves && t->total > 0) || !aligned_to(d_moves, 4))
        return fail(CX_ERR_INVALID, "cx_adamw_apply: null or misaligned moves");
    if (!d_lr && !(lr >= 0.0 && std::isfinite((float)lr)))
        return fail(CX_ERR_INVALID, "cx_adamw_apply: the learning rate must be finite and not negative");
    if (!(weight_decay >= 0.0 && std::isfinite((float)weight_decay)) || !std::isfinite((float)scale))
        return fail(CX_ERR_INVALID, "cx_adamw_apply: weight decay and scale must be finite, the former not negative");
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_adamw_apply(h, t, d_moves, (float)scale, lr, d_lr, weight_decay);
}

int cx_adamw_states(cx_handle h, cx_tensors t, cx_dtype dt, void* d_exp_avg, void* d_exp_avg_sq) {
    const int rc = check_set(h, t, "cx_adamw_states");
    if (rc != CX_OK) return rc;
    if (!t->adamw || t->state_bits != 8) return fail(CX_ERR_INVALID, "cx_adamw_states: the set has no 8-bit states");
    if (!number_type(dt)) return fail(CX_ERR_INVALID, "cx_adamw_states: values are fp32, bf16 or fp16");
    if (t->total > 0 && (!d_exp_avg || !d_exp_avg_sq || !aligned_to(d_exp_avg, element_bytes(dt)) ||
                         !aligned_to(d_exp_avg_sq, element_bytes(dt))))
        return fail(CX_ERR_INVALID, "cx_adamw_states: null or misaligned output");
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_adamw_states(h, t, dt, d_exp_avg, d_exp_avg_sq);
}

int cx_adamw_set_states(cx_handle h, cx_tensors t, const float* d_exp_avg, const float* d_exp_avg_sq) {
    const int rc = check_set(h, t, "cx_adamw_set_states");
    if (rc != CX_OK) return rc;
    if (!t->adamw || t->state_bits != 8) return fail(CX_ERR_INVALID, "cx_adamw_set_states: the set has no 8-bit states");
    if (t->total > 0 && (!d_exp_avg || !d_exp_avg_sq || !aligned_to(d_exp_avg, 4) || !aligned_to(d_exp_avg_sq, 4)))
        return fail(CX_ERR_INVALID, "cx_adamw_set_states: null or misaligned input");
    DeviceScope on(t->device);
    CX_HIP(on.error);
    return launch_adamw_set_states(h, t, d_exp_avg, d_exp_avg_sq);
}

}  // extern "C"
