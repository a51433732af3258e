// The kernel walk's stand-in for <hip/hip_runtime.h> with launches that are looked at instead of run, and the few builtins more that
// the sorting and scanning kernels need to compile: test infrastructure, never part of the library.
#pragma once
#define launch run_on_the_cpu
#include "../../kernel_walk/hip/hip_runtime.h"
#undef launch

inline unsigned long long __ballot(int) { return 0; }
inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
inline int __any(int v) { return v; }
inline unsigned atomicAdd(unsigned* p, unsigned v) { const unsigned o = *p; *p += v; return o; }
inline float __uint_as_float(uint32_t v) { float f; memcpy(&f, &v, 4); return f; }
inline uint32_t __float_as_uint(float f) { uint32_t v; memcpy(&v, &f, 4); return v; }
inline double __longlong_as_double(long long v) { double f; memcpy(&f, &v, 8); return f; }
inline long long __double_as_longlong(double f) { long long v; memcpy(&v, &f, 8); return v; }
inline int __double2hiint(double f) { return (int)(__double_as_longlong(f) >> 32); }
#define __hip_atomic_store(p, v, order, scope) (*(p) = (v))
#define __hip_atomic_load(p, order, scope) (*(p))
#define __HIP_MEMORY_SCOPE_AGENT 0
#define __builtin_amdgcn_s_sleep(x) ((void)0)

namespace fxemu {
inline const char* g_too_large = nullptr;  // why the last call's launch could not run
// The device's limits: fewer than 2^32 threads along x, 65535 blocks along y and z, 160 KB of LDS.
template <class F> inline void launch(dim3 grid, dim3 block, size_t smem_bytes, F&&) {
    ++g_launches;
    if (grid.x == 0 || grid.y == 0 || grid.z == 0) g_too_large = "an empty grid";
    if ((unsigned long long)grid.x * block.x >= 1ull << 32) g_too_large = "2^32 threads or more along x";
    if (grid.y > 65535 || grid.z > 65535) g_too_large = "more than 65535 blocks along y or z";
    if (smem_bytes > 160 * 1024) g_too_large = "more than 160 KB of LDS";
}
}  // namespace fxemu
