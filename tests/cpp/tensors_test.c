/* The calls over many tensors from plain C, with nothing but the library itself: a set, the gradients'
 * norms and clip coefficient, packing, an AdamW step on moments in 32 bits and the same in two halves, one on
 * moments in 8 bits, against the formulas in double, and the status codes of the error paths.  Prints the
 * PASSED / FAILED line of the other tests. */
#include <comprex_gfx950.h>

#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int errors = 0;
#define CHECK(cond)                                                         \
    do {                                                                    \
        if (!(cond)) {                                                      \
            printf("line %d: %s  [%s]\n", __LINE__, #cond, cx_last_error()); \
            ++errors;                                                       \
        }                                                                   \
    } while (0)

enum { N0 = 5000, N1 = 77, N = N0 + N1, B = 21 /* blocks of 256: 20 and 1 */ };

static cx_handle h;

static void* device(const void* from, size_t bytes) {
    void* p = NULL;
    CHECK(cx_device_alloc(&p, bytes) == CX_OK);
    CHECK(cx_copy(h, p, from, bytes) == CX_OK);
    return p;
}

/* one step of an element: everything in double */
static void formula(double* w, double* m, double* v, double g, double lr, double wd, int t) {
    *m = 0.9 * *m + 0.1 * g;
    *v = 0.999 * *v + 0.001 * g * g;
    *w -= lr * wd * *w + lr / (1 - pow(0.9, t)) * *m / (sqrt(*v) / sqrt(1 - pow(0.999, t)) + 1e-8);
}

/* roundings to fp32 along the way: below 20 of the weight and 40 of the move, which is at most 4 lr here */
static int near(double got, double want, double lr) { return fabs(got - want) <= 0x1p-24 * (20 * fabs(want) + 160 * lr); }

/* a double rounded to fp32 once, summed in another order before */
static int rounded(float got, double want) { return fabs(got - want) <= 0x1.001p-24 * want; }

int main(void) {
    if (cx_device_count() < 1) {
        printf("no GPU: this test drives the HIP library and cannot run here\n");
        return 77;
    }
    static float w[N], g[N], zero[N], got[N], flat[N], moves[N];
    unsigned x = 7u;
    for (int i = 0; i < N; ++i) {
        x = x * 1664525u + 1013904223u;
        w[i] = (float)((int)((x >> 8) % 20001u) - 10000) / 8192.0f;
        x = x * 1664525u + 1013904223u;
        g[i] = (float)((int)((x >> 8) % 20001u) - 10000) / 65536.0f;
    }
    CHECK(cx_create(&h, NULL) == CX_OK);
    float *d_w = device(w, sizeof w), *d_g = device(g, sizeof g), *d_m = device(zero, sizeof zero), *d_v = device(zero, sizeof zero);
    float *d_flat = device(zero, sizeof zero), *d_norms = device(zero, 16), *d_coef = device(zero, 4);
    int* d_bad = device(zero, 4);
    const long long sizes[2] = {N0, N1};
    void *params[2] = {d_w, d_w + N0}, *ms[2] = {d_m, d_m + N0}, *vs[2] = {d_v, d_v + N0};
    cx_adamw_state state = {CX_F32, 32, params, NULL, ms, vs, NULL, NULL};
    cx_tensors set = NULL;
    CHECK(cx_tensors_create(&set, h, 2, sizes, &state) == CX_OK);

    const void* each[2] = {d_g, d_g + N0};
    cx_grads grads = {CX_F32, each, NULL}, as_flat = {CX_F32, NULL, d_g};
    float norms[3], coef = 0;
    int bad = 7;
    double s0 = 0, s1 = 0;
    for (int i = 0; i < N; ++i) *(i < N0 ? &s0 : &s1) += (double)g[i] * g[i];
    CHECK(cx_grad_norms(h, set, &grads, 1.0, 1.0, 0, d_norms, d_coef, d_bad) == CX_OK);
    CHECK(cx_copy(h, norms, d_norms, 12) == CX_OK && cx_copy(h, &coef, d_coef, 4) == CX_OK && cx_copy(h, &bad, d_bad, 4) == CX_OK);
    CHECK(rounded(norms[0], sqrt(s0)) && rounded(norms[1], sqrt(s1)) && rounded(norms[2], sqrt(s0 + s1)) && bad == 0);
    CHECK(rounded(coef, 1.0 / sqrt(s0 + s1)));
    CHECK(cx_pack(h, set, &grads, d_coef, 1, 2.0, d_bad, d_flat) == CX_OK);
    CHECK(cx_copy(h, flat, d_flat, sizeof flat) == CX_OK);
    for (int i = 0; i < N; ++i)
        if (flat[i] != g[i] * (coef * 2.0f)) CHECK(!"packed");

    /* three steps; the last one in two halves */
    static double ww[N], mm[N], vv[N];
    for (int i = 0; i < N; ++i) ww[i] = w[i];
    const double lr = 0x1p-6, wd = 0.1;
    cx_adamw_args a = {lr, 0.9, 0.999, 1e-8, wd, 1.0, 0, NULL, NULL, d_coef, 1, d_bad, NULL};
    for (int t = 1; t <= 3; ++t) {
        a.step = t;
        a.d_moves = t == 3 ? d_flat : NULL;
        CHECK(cx_adamw_step(h, set, t == 2 ? &as_flat : &grads, &a) == CX_OK);
        if (t == 3) CHECK(cx_adamw_apply(h, set, d_flat, 1.0, lr, NULL, wd) == CX_OK);
        CHECK(cx_copy(h, got, d_w, sizeof got) == CX_OK);
        for (int i = 0; i < N; ++i) {
            formula(&ww[i], &mm[i], &vv[i], (double)g[i] * coef, lr, wd, t);
            if (!near(got[i], ww[i], t * lr)) CHECK(!"step");
        }
    }

    /* moments in 8 bits: a first step moves by lr (1 - eps / |g|), whatever the rounding behind it */
    static unsigned char no_bytes[N];
    unsigned char *d_m8 = device(no_bytes, N), *d_v8 = device(no_bytes, N);
    float *d_ms = device(zero, B * 4), *d_vs = device(zero, B * 4), *d_m32 = device(zero, sizeof zero), *d_v32 = device(zero, sizeof zero);
    void *m8[2] = {d_m8, d_m8 + N0}, *v8[2] = {d_v8, d_v8 + N0};
    float *scales_m[2] = {d_ms, d_ms + 20}, *scales_v[2] = {d_vs, d_vs + 20};
    cx_adamw_state small = {CX_F32, 8, params, NULL, m8, v8, scales_m, scales_v};
    cx_tensors set8 = NULL;
    CHECK(cx_tensors_create(&set8, h, 2, sizes, &small) == CX_OK);
    CHECK(cx_copy(h, d_w, w, sizeof w) == CX_OK);
    a.step = 1;
    a.d_moves = NULL;
    CHECK(cx_adamw_step(h, set8, &grads, &a) == CX_OK);
    CHECK(cx_copy(h, got, d_w, sizeof got) == CX_OK);
    CHECK(cx_adamw_states(h, set8, CX_F32, d_m32, d_v32) == CX_OK);
    CHECK(cx_copy(h, moves, d_m32, sizeof moves) == CX_OK);
    for (int i = 0; i < N; ++i) {
        double wi = w[i], mi = 0, vi = 0;
        formula(&wi, &mi, &vi, (double)g[i] * coef, lr, wd, 1);
        if (!near(got[i], wi, lr)) CHECK(!"8-bit step");
        if (fabs(moves[i] - mi) > fabs(mi) * 0.0626 + 2e-7) CHECK(!"8-bit moment");  /* half a step; the block's smallest */
    }
    CHECK(cx_adamw_set_states(h, set8, d_m32, d_v32) == CX_OK);

    /* what is refused leaves a text, and nothing changes */
    cx_tensors other = NULL;
    void* twice[2] = {d_w, d_w + 10};
    cx_adamw_state overlap = {CX_F32, 32, twice, NULL, ms, vs, NULL, NULL};
    CHECK(cx_tensors_create(&other, h, 2, sizes, &overlap) == CX_ERR_INVALID && !other && strlen(cx_last_error()) > 0);
    CHECK(cx_adamw_states(h, set, CX_F32, d_m32, d_v32) == CX_ERR_INVALID);
    CHECK(cx_adamw_step(h, set, &grads, NULL) == CX_ERR_INVALID);
    a.n_coefs = 3;
    CHECK(cx_adamw_step(h, set, &grads, &a) == CX_ERR_SIZE_MISMATCH);
    a.n_coefs = 1;
    a.step = 0;
    CHECK(cx_adamw_step(h, set, &grads, &a) == CX_ERR_INVALID);
    cx_grads both = {CX_F32, each, d_g}, none = {CX_F32, NULL, NULL}, doubles = {CX_F64, each, NULL};
    CHECK(cx_pack(h, set, &both, NULL, 0, 1.0, NULL, d_flat) == CX_ERR_INVALID);
    CHECK(cx_pack(h, set, &none, NULL, 0, 1.0, NULL, d_flat) == CX_ERR_INVALID);
    CHECK(cx_pack(h, set, &doubles, NULL, 0, 1.0, NULL, d_flat) == CX_ERR_INVALID);
    CHECK(cx_pack(h, set, &as_flat, NULL, 0, 1.0, NULL, d_g + 1) == CX_ERR_INVALID);
    CHECK(cx_grad_norms(h, set, &grads, 1.0, 0.0, 0, d_norms, d_coef, d_bad) == CX_ERR_INVALID);
    CHECK(cx_tensors_create(&other, h, 0, NULL, NULL) == CX_OK && cx_tensors_destroy(other) == CX_OK);

    CHECK(cx_synchronize(h) == CX_OK);
    CHECK(cx_tensors_destroy(set) == CX_OK && cx_tensors_destroy(set8) == CX_OK);
    void* all[] = {d_w, d_g, d_m, d_v, d_flat, d_norms, d_coef, d_bad, d_m8, d_v8, d_ms, d_vs, d_m32, d_v32};
    for (unsigned i = 0; i < sizeof all / sizeof *all; ++i) CHECK(cx_device_free(all[i]) == CX_OK);
    CHECK(cx_destroy(h) == CX_OK);
    printf("calls over many tensors from plain C\n");
    if (errors == 0) printf("+++ PASSED +++\n");
    else printf("--- FAILED ---\nwith %d errors.\n", errors);
    return errors ? 1 : 0;
}
