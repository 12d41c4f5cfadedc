// TEST INFRASTRUCTURE ONLY: the host builtins of the device prelude and, beside them, those that the operators of a
// decoding step use.  As there, one thread runs at a time: lane exchanges return the caller's own value.
#pragma once
#include "../../host_builtins.h"
#define MONONN_ONE_THREAD
#define MONONN_KEEP_IN_VGPR(v) ((void)0)
typedef short mononn_short4 __attribute__((ext_vector_type(4)));
inline mononn_short4 host_lds_read8(const char* p) {
  mononn_short4 v;
  std::memcpy(&v, p, 8);
  return v;
}
#define MONONN_LDS_READ_TR16(p) host_lds_read8(p)
inline void sincospif(float x, float* s, float* c) { *s = sinf(3.14159265f * x), *c = cosf(3.14159265f * x); }
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_s_setprio(p) ((void)0)
#define __any(x) (x)
#define __all(x) (x)
#define __ballot(x) ((x) ? 1ull : 0ull)
#define __shfl(v, ...) (v)
#define __builtin_amdgcn_readlane(v, l) (v)
#define __shfl_up(v, ...) (v)
struct HostPair {
  unsigned v[2];
  unsigned operator[](int i) const { return v[i]; }
};
inline HostPair host_swap(unsigned a, unsigned b) { return {{b, a}}; }
#define __builtin_amdgcn_permlane32_swap(a, b, x, y) host_swap(a, b)
#define __builtin_amdgcn_permlane16_swap(a, b, x, y) host_swap(a, b)
