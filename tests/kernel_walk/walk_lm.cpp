// CPU walk of the language-model kernels whose addresses do not depend on loaded data: test infrastructure, a sibling of walk_gemm.cpp.
// -DWALK_GEMM: gemm.hip's products with the whole epilogue (bias, activation, residual, pre-activation); -DWALK_NORM: rmsnorm.hip;
// -DWALK_ACT: linear_act.hip (its product calls are stubs here).  Every thread of every launch runs on the CPU; every tensor and the
// library scratch are buffers of exactly their size between inaccessible pages, once with the END of each against a guard page and
// once with the START.
//
// usage: walk_lm < cases    with one case per line:
//   <name> <f32|f64> <a> <b> <c> <shift>     products: M N K; norm: rows dim -; act: rows out -; tensors start `shift` elements into a
//                                            16-byte block (the library itself only needs element alignment)
#define FX_HOST_EMULATION 1
#if defined(WALK_GEMM)
#include "../../ferrox_amd/csrc/gemm.hip"
#elif defined(WALK_NORM)
#include "../../ferrox_amd/csrc/rmsnorm.hip"
#else
#include "../../ferrox_amd/csrc/linear_act.hip"
#endif

#include <csignal>
#include <iostream>
#include <sstream>
#include <string>

namespace fx {
void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfprintf(stderr, fmt, ap);
    fputc('\n', stderr);
    va_end(ap);
}
int bind_device(int) { return FX_OK; }
}  // namespace fx
#if defined(WALK_GEMM)
extern "C" int fx_bias_act_f32(fx_ctx*, float*, const float*, int64_t, int64_t, int64_t, int) { return FX_OK; }
extern "C" int fx_bias_act_f64(fx_ctx*, double*, const double*, int64_t, int64_t, int64_t, int) { return FX_OK; }
extern "C" int fx_bias_grad_f32(fx_ctx*, const float*, float*, int64_t, int64_t, int64_t) { return FX_OK; }
extern "C" int fx_bias_grad_f64(fx_ctx*, const double*, double*, int64_t, int64_t, int64_t) { return FX_OK; }
extern "C" int fx_relu_bwd_f32(fx_ctx*, const float*, const float*, float*, int64_t) { return FX_OK; }
extern "C" int fx_relu_bwd_f64(fx_ctx*, const double*, const double*, double*, int64_t) { return FX_OK; }
#elif defined(WALK_NORM)
extern "C" int fx_fill_f32(fx_ctx*, float*, float, int64_t) { return FX_OK; }
extern "C" int fx_fill_f64(fx_ctx*, double*, double, int64_t) { return FX_OK; }
#else
extern "C" int fx_linear_bwd_f32(fx_ctx*, int64_t, int64_t, int64_t, const float*, const float*, const float*, float*, float*, float*, int) { return FX_OK; }
extern "C" int fx_linear_bwd_f64(fx_ctx*, int64_t, int64_t, int64_t, const double*, const double*, const double*, double*, double*, double*, int) {
    return FX_OK;
}
#endif

static fxemu::GuardedBuffer g_scratch;
void* fx_ctx::get_scratch(i64 bytes) {
    g_scratch.reset((size_t)bytes, fxemu::g_at_end);
    return g_scratch.ptr;
}

namespace {
std::string g_case;
const char* g_short = "";  // the detector's self-test: this tensor is one element too short
struct Buf {
    fxemu::GuardedBuffer b;
    // `elems` elements that end (or, in the other pass, start) at the guard; the start is `shift` elements behind a 16-byte border
    template <typename T> T* get(i64 elems, int shift, const char* name = "") {
        if (*name && strcmp(name, g_short) == 0) --elems;
        const size_t bytes = (size_t)elems * sizeof(T), lead = (size_t)shift * sizeof(T);
        if (!fxemu::g_at_end) {
            b.reset(bytes + lead, false);
            return reinterpret_cast<T*>(b.ptr + lead);
        }
        b.reset(bytes + 32, true);
        // the end against the guard when the size allows the alignment asked for, else up to 15 bytes in front of it
        char* p = b.ptr + 32;
        p -= ((uintptr_t)p - lead) & 15;
        return reinterpret_cast<T*>(p);
    }
};
void on_fault(int) {
    const char* a = "\nFAULT (signal) while walking: ";
    (void)!write(2, a, strlen(a));
    (void)!write(2, g_case.c_str(), g_case.size());
    (void)!write(2, "\n", 1);
    _exit(3);
}
void check(int rc, const char* what) {
    if (rc != FX_OK) {
        fprintf(stderr, "%s returned %d for %s\n", what, rc, g_case.c_str());
        exit(4);
    }
}

#if defined(WALK_GEMM)
int call(fx_ctx* c, int ta, int tb, i64 M, i64 N, i64 K, const float* A, const float* B, const float* b, const float* r, float* p, float* C, int act) {
    return fx_gemm_bias_act_residual_f32(c, ta, tb, M, N, K, A, B, b, r, p, C, act);
}
int call(fx_ctx* c, int ta, int tb, i64 M, i64 N, i64 K, const double* A, const double* B, const double* b, const double* r, double* p, double* C, int act) {
    return fx_gemm_bias_act_residual_f64(c, ta, tb, M, N, K, A, B, b, r, p, C, act);
}
template <typename T> void walk_case(fx_ctx* c, i64 M, i64 N, i64 K, int shift) {
    Buf ba, bb, bc, bbias, bres, bpre;
    // shift 2: the operands and C on their borders (as the slab tiles want them), the epilogue's tensors off it
    const int so = shift == 2 ? 0 : shift, se = shift == 2 ? 1 : shift;
    T *A = ba.get<T>(M * K, so), *B = bb.get<T>(K * N, so), *C = bc.get<T>(M * N, so, "c");
    T *bias = bbias.get<T>(N, se, "bias"), *res = bres.get<T>(M * N, se, "residual"), *pre = bpre.get<T>(M * N, se, "pre");
    for (int ta = 0; ta < 2; ++ta)
        for (int tb = 0; tb < 2; ++tb) {
            check(call(c, ta, tb, M, N, K, A, B, bias, res, pre, C, 1), "fx_gemm_bias_act_residual");
            check(call(c, ta, tb, M, N, K, A, B, bias, res, pre, C, 2), "fx_gemm_bias_act_residual (gelu)");
        }
}
#elif defined(WALK_NORM)
template <typename T> struct Norm;
template <> struct Norm<float> { static constexpr auto fwd = fx_rmsnorm_fwd_f32; static constexpr auto bwd = fx_rmsnorm_bwd_f32; };
template <> struct Norm<double> { static constexpr auto fwd = fx_rmsnorm_fwd_f64; static constexpr auto bwd = fx_rmsnorm_bwd_f64; };
template <typename T> void walk_case(fx_ctx* c, i64 rows, i64 D, i64, int shift) {
    Buf b[9];
    const i64 n = rows * D;
    T *x = b[0].get<T>(n, shift), *res = b[1].get<T>(n, shift, "residual"), *h = b[2].get<T>(n, shift), *y = b[3].get<T>(n, shift, "y");
    T *w = b[4].get<T>(D, shift, "w"), *r = b[5].get<T>(rows, 0), *dx = b[6].get<T>(n, shift), *dw = b[7].get<T>(D, shift, "dw");
    check(Norm<T>::fwd(c, x, nullptr, w, 1e-6, nullptr, y, r, rows, D), "fx_rmsnorm_fwd");
    check(Norm<T>::fwd(c, x, res, w, 1e-6, h, y, nullptr, rows, D), "fx_rmsnorm_fwd with residual");
    check(Norm<T>::bwd(c, x, nullptr, h, w, r, dx, dw, rows, D), "fx_rmsnorm_bwd");
    check(Norm<T>::bwd(c, x, res, h, w, r, dx, nullptr, rows, D), "fx_rmsnorm_bwd with dh");
}
#else
template <typename T> struct Act;
template <> struct Act<float> { static constexpr auto bwd = fx_linear_act_bwd_f32; };
template <> struct Act<double> { static constexpr auto bwd = fx_linear_act_bwd_f64; };
template <typename T> void walk_case(fx_ctx* c, i64 rows, i64 out, i64, int shift) {
    Buf b[8];
    T *dy = b[0].get<T>(rows * out, shift), *pre = b[1].get<T>(rows * out, shift, "pre"), *dpre = b[2].get<T>(rows * out, shift), *db = b[3].get<T>(out, shift, "db");
    T *W = b[4].get<T>(out, 0), *X = b[5].get<T>(rows, 0), *dX = b[6].get<T>(rows, 0), *dW = b[7].get<T>(out, 0);
    for (int act = 0; act < 4; ++act) check(Act<T>::bwd(c, rows, 1, out, dy, W, X, pre, act, dpre, dX, dW, act & 1 ? db : nullptr), "fx_linear_act_bwd");
    check(Act<T>::bwd(c, rows, 1, out, dy, W, X, pre, 2, dpre, dX, dW, db), "fx_linear_act_bwd");
    // the last vectors of a row of almost 2^31 elements, of which only the end is there
    constexpr int V = 16 / (int)sizeof(T), D = 0x7fffffff, LAST = D / V * V;
    Buf end;
    T* const tail = end.get<T>(D - LAST + V, 0);  // elements LAST - V .. D - 1
    T* const row = tail - (LAST - V);
    T v[V];
    for (int u = 0; u < D - LAST + V; ++u) tail[u] = T(u + 1);
    for (int j : {LAST - V, LAST}) {
        vio::load_part<V>(row, j, D, v);
        for (int u = 0; u < V; ++u)
            if (v[u] != (u < D - j ? T(j - (LAST - V) + u + 1) : T(0))) check(FX_ERR_INVALID, "load_part");
        vio::store_part<V>(row, j, D, v);
    }
}
#endif
}  // namespace

int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    if (const char* v = getenv("FX_WALK_SHORT")) g_short = v;
    fx_ctx ctx;
    ctx.device = 0;
    ctx.num_cus = 256;
    std::string line;
    int ncases = 0;
    while (std::getline(std::cin, line)) {
        if (line.empty()) continue;
        std::istringstream ss(line);
        std::string name, dt;
        i64 a, b, c;
        int shift;
        ss >> name >> dt >> a >> b >> c >> shift;
        if (!ss) {
            fprintf(stderr, "bad case line: %s\n", line.c_str());
            return 2;
        }
        for (int pass = 0; pass < 2; ++pass) {
            fxemu::g_at_end = pass == 0;
            g_case = line + (pass == 0 ? "  [ends exact]" : "  [starts exact]");
            if (dt == "f64") walk_case<double>(&ctx, a, b, c, shift);
            else walk_case<float>(&ctx, a, b, c, shift);
        }
        ++ncases;
    }
    printf("walked %d cases, %llu launches: every access stayed inside its buffer\n", ncases, fxemu::g_launches);
    return 0;
}
