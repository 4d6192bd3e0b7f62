// Host restatement of apex_amd/csrc/gfx950/half_types.h: the conversions in integer arithmetic, the fast instructions as libm's functions.  Test infrastructure only.
#pragma once
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>

namespace half_types {

inline float widen_bf16(uint16_t u) { return hipemu::asf((uint32_t)u << 16); }
inline uint16_t round_bf16(float x) {
    const uint32_t u = hipemu::asu(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);      // NaN stays NaN
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
inline float widen_f16(uint16_t h) {
    const uint32_t s = (uint32_t)(h & 0x8000u) << 16, e = (h >> 10) & 31u, m = h & 1023u;
    if (e == 31) return hipemu::asf(s | 0x7f800000u | (m << 13));
    const float v = e ? ldexpf((float)(m | 1024u), (int)e - 25) : ldexpf((float)m, -24);
    return s ? -v : v;
}
inline uint16_t round_f16(float x) {
    const uint32_t u = hipemu::asu(x), s = (u >> 16) & 0x8000u;
    const float a = fabsf(x);
    if (a != a) return (uint16_t)(s | 0x7e00u);
    if (a >= 65520.f) return (uint16_t)(s | 0x7c00u);
    int e = a < 6.103515625e-05f ? -24 : ilogbf(a) - 10;                             // exponent of the last bit
    const float q = nearbyintf(ldexpf(a, -e));                                       // 0 .. 2048, to nearest even
    uint32_t m = (uint32_t)q;
    if (e == -24) return (uint16_t)(s | m);                                          // (1024: the smallest normal number, its own code)
    if (m == 2048u) { m = 1024u; ++e; }
    return (uint16_t)(s | ((uint32_t)(e + 25) << 10) | (m - 1024u));
}
inline float exp2_fast(float x) { return exp2f(x); }
inline float rcp_fast(float x) { return 1.0f / x; }
inline float sqrt_fast(float x) { return sqrtf(x); }

#define APX_PASSING(p) (*(p))
#define APX_PASS(p, x) (*(p) = (x))
inline int wave_uniform(int x) { return x; }
inline unsigned lane_offset(unsigned x) { return x; }
#define APX_GLOBAL
template <class T> inline T* wave_address(T* p) { return p; }

}  // namespace half_types
