// esda_softcap.h -- scores capped by a tanh, for the sources of esda_scored.h's entry points.
#pragma once

#include <cmath>

// s = cap tanh(x / cap), x = scale q.k, in log2 units from raw = q.k.
//
// With e = 2^(in raw) = e^(2 x / cap), tanh is 1 - 2 / (1 + e): an exponential and a reciprocal, but
// off by up to 2^-22 whatever its size, so the score by cap 2^-21.  Up to kNarrowCap that is 2^-13 of a
// weight, a sixteenth of its rounding to bf16.  Wider caps (wide) take the quotient of tanh's continued
// fraction at its fifth term where |x| < cap,
//   tanh y = y (945 + 105 y^2 + y^4) / (945 + 420 y^2 + 15 y^4)   (within 2^-23 of itself for |y| <= 1),
// which leaves s off by 2^-21 of s: x itself where the cap is far away.
struct SoftCap {
    float in, out, y;  // 2 log2 e scale / cap; cap log2 e, or 0: no cap; scale / cap
    int wide;
};

constexpr float kNarrowCap = 256.0f;

// Fills c for a cap >= 0; false where fp32 cannot hold its factors.
inline bool set_softcap(float cap, float scale, SoftCap *c) {
    *c = SoftCap{};
    if (cap == 0.0f) return true;
    c->in = (float) (2.0 * 1.4426950408889634 * scale / cap);
    c->out = (float) (1.4426950408889634 * cap);
    c->y = (float) ((double) scale / cap);
    c->wide = cap > kNarrowCap;
    return std::isfinite(c->in) && std::isfinite(c->out) && c->in != 0.0f;
}

#if defined(__HIP__)
__device__ __forceinline__ float capped_narrow(float raw, const SoftCap &c) {
    return c.out * __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(raw * c.in)), 1.0f);
}
// x: the score without a cap, log2 units
__device__ __forceinline__ float capped_wide(float raw, float x, const SoftCap &c) {
    const float y = raw * c.y, t = y * y;
    const float num = __builtin_fmaf(t, t + 105.0f, 945.0f), den = __builtin_fmaf(t, __builtin_fmaf(15.0f, t, 420.0f), 945.0f);
    const float near = x * (num * __builtin_amdgcn_rcpf(den));
    return t < 1.0f ? near : capped_narrow(raw, c);
}
#endif
