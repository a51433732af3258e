// Calls of the language-model operators with sizes that no test could hold in memory: what each would launch is held against the
// device's limits (hip/hip_runtime.h beside this file), nothing runs and no pointer is followed.  Test infrastructure.
//
// usage: limits < cases    with one case per line:  <call> <f32|f64> <sizes ...>
// prints per case:  <launches> launches | refused: <message> | TOO LARGE: <why>
#define FX_HOST_EMULATION 1
#if defined(LIMITS_GEMM)
#include "../../ferrox_amd/csrc/gemm.hip"
#elif defined(LIMITS_NORM)
#include "../../ferrox_amd/csrc/rmsnorm.hip"
#elif defined(LIMITS_ACT)
#include "../../ferrox_amd/csrc/linear_act.hip"
#elif defined(LIMITS_EMBED)
#include "../../ferrox_amd/csrc/embedding.hip"
#elif defined(LIMITS_SCAN)
#include "../../ferrox_amd/csrc/recurrence.hip"
#else
#include "../../ferrox_amd/csrc/gradnorm.hip"
#endif

#include <iostream>
#include <sstream>
#include <string>

static char g_message[512];
namespace fx {
void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_message, sizeof(g_message), fmt, ap);
    va_end(ap);
}
int bind_device(int) { return FX_OK; }
}  // namespace fx

// tensors 2^44 bytes apart
static char* at(int k) { return reinterpret_cast<char*>((uintptr_t)(k + 1) << 44); }
void* fx_ctx::get_scratch(i64) { return at(40); }
template <typename T> static T* tensor(int k) { return reinterpret_cast<T*>(at(k)); }

#if defined(LIMITS_GEMM)
extern "C" int fx_bias_act_f32(fx_ctx*, float*, const float*, int64_t, int64_t, int64_t, int) { return FX_OK; }
extern "C" int fx_bias_act_f64(fx_ctx*, double*, const double*, int64_t, int64_t, int64_t, int) { return FX_OK; }
extern "C" int fx_bias_grad_f32(fx_ctx*, const float*, float*, int64_t, int64_t, int64_t) { return FX_OK; }
extern "C" int fx_bias_grad_f64(fx_ctx*, const double*, double*, int64_t, int64_t, int64_t) { return FX_OK; }
extern "C" int fx_relu_bwd_f32(fx_ctx*, const float*, const float*, float*, int64_t) { return FX_OK; }
extern "C" int fx_relu_bwd_f64(fx_ctx*, const double*, const double*, double*, int64_t) { return FX_OK; }
#elif defined(LIMITS_NORM)
extern "C" int fx_fill_f32(fx_ctx*, float*, float, int64_t) { return FX_OK; }
extern "C" int fx_fill_f64(fx_ctx*, double*, double, int64_t) { return FX_OK; }
#elif defined(LIMITS_ACT)
extern "C" int fx_linear_bwd_f32(fx_ctx*, int64_t, int64_t, int64_t, const float*, const float*, const float*, float*, float*, float*, int) { return FX_OK; }
extern "C" int fx_linear_bwd_f64(fx_ctx*, int64_t, int64_t, int64_t, const double*, const double*, const double*, double*, double*, double*, int) {
    return FX_OK;
}
#endif

template <typename T> int call(fx_ctx* c, const std::string& what, i64 a, i64 b, i64 d) {
    constexpr bool S = sizeof(T) == 4;
    T* t[10];
    for (int k = 0; k < 10; ++k) t[k] = tensor<T>(k);
    int64_t* const ids = tensor<int64_t>(20);
    (void)ids;
#define CALL(name, ...) (([&](auto* f32, auto* f64) { if constexpr (S) return f32(__VA_ARGS__); else return f64(__VA_ARGS__); })(name##_f32, name##_f64))
#if defined(LIMITS_GEMM)
    if (what == "linear") return CALL(fx_gemm_bias_act_residual, c, 0, 1, a, b, d, t[0], t[1], t[2], t[3], t[4], t[5], 2);
#elif defined(LIMITS_NORM)
    if (what == "norm") return CALL(fx_rmsnorm_fwd, c, t[0], (const T*)nullptr, t[1], 1e-6, (T*)nullptr, t[0], t[2], a, b);
    if (what == "norm_res") return CALL(fx_rmsnorm_fwd, c, t[0], t[3], t[1], 1e-6, t[3], t[0], t[2], a, b);
    if (what == "norm_bwd") return CALL(fx_rmsnorm_bwd, c, t[0], t[1], t[2], t[3], t[4], t[0], t[5], a, b);
#elif defined(LIMITS_ACT)
    if (what == "act_bwd") return CALL(fx_linear_act_bwd, c, a, 1, b, t[0], t[1], t[2], t[3], 2, t[0], t[4], t[5], t[6]);
#elif defined(LIMITS_EMBED)
    if (what == "embed") return CALL(fx_embedding_fwd, c, t[0], ids, t[1], a, b, d, T(1));
    if (what == "embed_bwd") return CALL(fx_embedding_bwd, c, t[0], ids, t[1], a, b, d, T(1));
#elif defined(LIMITS_SCAN)
    if (what == "scan") return CALL(fx_gated_recurrence_fwd, c, t[0], t[1], t[2], t[3], a, b, d);
    if (what == "scan_bwd") return CALL(fx_gated_recurrence_bwd, c, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], a, b, d);
#else
    if (what == "clip") {  // a tensors of b elements
        std::vector<T*> g;
        std::vector<int64_t> n((size_t)a, b);
        for (i64 k = 0; k < a; ++k) g.push_back(tensor<T>(0) + k * b);
        return CALL(fx_clip_grad_norm_multi, c, (int)a, g.data(), g.data(), n.data(), 1.0, tensor<T>(20));
    }
#endif
    fprintf(stderr, "no call %s\n", what.c_str());
    exit(2);
}

int main() {
    fx_ctx ctx;
    ctx.num_cus = 256;
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream ss(line);
        std::string what, dt;
        i64 a, b, d;
        ss >> what >> dt >> a >> b >> d;
        fxemu::g_launches = 0;
        fxemu::g_too_large = nullptr;
        const int rc = dt == "f64" ? call<double>(&ctx, what, a, b, d) : call<float>(&ctx, what, a, b, d);
        if (fxemu::g_too_large) printf("TOO LARGE: %s\n", fxemu::g_too_large);
        else if (rc != FX_OK) printf("refused: %s\n", g_message);
        else printf("%llu launches\n", fxemu::g_launches);
    }
    return 0;
}
