// A gated linear recurrence over time-major sequences [T, B, H], its backward pass and its one-step form (include/apx.h, apx_gated_scan_*).
//
//   a = sigmoid(f), n = 1 - a;   p_t = reset ? 0 : h_{t-1};   h_t = a_t p_t + n_t x_t;   y_t = h_t sigmoid(o_t)
//   backward, c_{T-1} = dh_last:  g_t = dy_t sigmoid(o_t) + c_t;   c_{t-1} = reset ? 0 : a_t g_t;   dh0 = c_{-1}
//     dx_t = n_t g_t     df_t = g_t (p_t - x_t) a_t n_t     do_t = dy_t h_t s (1 - s), s = sigmoid(o_t)
//
// The channels (b, j) are independent of each other.  The backward pass needs every h_t again: the forward pass keeps the state in front of every 16th step (1/16 of the
// states, f32), and the steps between are run again from there.
#include "apx_common.h"
#include <gfx950/half_types.h>

namespace {

using namespace half_types;

template <int TYPE> struct Elem;
template <> struct Elem<APX_F32> {
    typedef float raw;
    static __device__ __forceinline__ float get(raw r) { return r; }
    static __device__ __forceinline__ raw put(float v) { return v; }
};
template <> struct Elem<APX_BF16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float get(raw r) { return widen_bf16(r); }
    static __device__ __forceinline__ raw put(float v) { return round_bf16(v); }
};
template <> struct Elem<APX_F16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float get(raw r) { return widen_f16(r); }
    static __device__ __forceinline__ raw put(float v) { return round_f16(v); }
};

constexpr int KEEP = 16;                  // steps between two kept states
constexpr float LOG2E = 1.44269504088896340736f;

// a = sigmoid(f) and n = 1 - a.  Whichever is below 1/2 is formed without cancellation, the other as 1 minus it, so that a + n = 1 to the last bit of the larger one: what
// a long memory loses and what it takes in stay in balance whatever the errors of the fast exponential and reciprocal.  f = +-inf gives exactly 1 and 0, a NaN two of them.
__device__ __forceinline__ void gate(float f, float& a, float& n) {
    const float e = exp2_fast(-fabsf(f) * LOG2E);
    const float lo = e * rcp_fast(1.f + e), hi = 1.f - lo;
    a = f >= 0.f ? hi : lo;
    n = f >= 0.f ? lo : hi;
}
__device__ __forceinline__ float sigmoid(float f) { float a, n; gate(f, a, n); return a; }

struct Strides { int64_t t, b; };
struct Scan {
    int64_t T, B; int H;
    const void *f, *x, *o, *dy; void *y, *df, *dx, *do_;
    Strides sf, sx, so, sy, sdy, sdf, sdx, sdo;
    const float *h0, *dh_last; float *h_last, *save, *dh0;
    const uint8_t* reset; const int32_t* lens;
};

template <int TYPE>
__global__ __launch_bounds__(64) void gated_scan_fwd_kernel(Scan S) {
    typedef Elem<TYPE> E; typedef typename E::raw raw;
    const int64_t c = blockIdx.x * (int64_t)64 + threadIdx.x, BH = S.B * S.H;
    if (c >= BH) return;
    const int64_t b = c / S.H; const int j = (int)(c - b * S.H);
    const int64_t len = S.lens ? S.lens[b] : S.T;
    const raw* f = (const raw*)S.f + b * S.sf.b + j; const raw* x = (const raw*)S.x + b * S.sx.b + j;
    const raw* o = S.o ? (const raw*)S.o + b * S.so.b + j : nullptr;
    raw* y = (raw*)S.y + b * S.sy.b + j;
    float h = S.h0 ? S.h0[c] : 0.f;
    for (int64_t t = 0; t < S.T; ++t) {
        if (S.save && t % KEEP == 0) S.save[(t / KEEP) * BH + c] = h;
        float out = 0.f;
        if (t < len) {
            float a, n;
            gate(E::get(f[t * S.sf.t]), a, n);
            const float v = n * E::get(x[t * S.sx.t]);
            h = S.reset && S.reset[t * S.B + b] ? v : fmaf(a, h, v);
            out = o ? h * sigmoid(E::get(o[t * S.so.t])) : h;
        }
        y[t * S.sy.t] = E::put(out);
    }
    S.h_last[c] = h;
}

template <int TYPE>
__global__ __launch_bounds__(64) void gated_scan_bwd_kernel(Scan S) {
    typedef Elem<TYPE> E; typedef typename E::raw raw;
    const int64_t c = blockIdx.x * (int64_t)64 + threadIdx.x, BH = S.B * S.H;
    if (c >= BH) return;
    const int64_t b = c / S.H; const int j = (int)(c - b * S.H);
    const int64_t len = S.lens ? S.lens[b] : S.T;
    const raw* f = (const raw*)S.f + b * S.sf.b + j; const raw* x = (const raw*)S.x + b * S.sx.b + j;
    const raw* o = S.o ? (const raw*)S.o + b * S.so.b + j : nullptr; const raw* dy = (const raw*)S.dy + b * S.sdy.b + j;
    raw* df = (raw*)S.df + b * S.sdf.b + j; raw* dx = (raw*)S.dx + b * S.sdx.b + j; raw* dO = o ? (raw*)S.do_ + b * S.sdo.b + j : nullptr;
    float carry = S.dh_last ? S.dh_last[c] : 0.f;
    for (int64_t k = (S.T + KEEP - 1) / KEEP - 1; k >= 0; --k) {
        const int64_t t0 = k * KEEP;
        float prev[KEEP];
        float h = S.save[k * BH + c];
        for (int i = 0; i < KEEP; ++i) {
            const int64_t t = t0 + i;
            if (t >= len || t >= S.T) continue;
            if (S.reset && S.reset[t * S.B + b]) h = 0.f;
            prev[i] = h;
            float a, n;
            gate(E::get(f[t * S.sf.t]), a, n);
            h = fmaf(a, h, n * E::get(x[t * S.sx.t]));
        }
        for (int i = KEEP - 1; i >= 0; --i) {
            const int64_t t = t0 + i;
            if (t >= S.T) continue;
            float gf = 0.f, gx = 0.f, go = 0.f;
            if (t < len) {
                float a, n;
                gate(E::get(f[t * S.sf.t]), a, n);
                const float xv = E::get(x[t * S.sx.t]), d = E::get(dy[t * S.sdy.t]);
                float g = d + carry;
                if (o) {
                    float s, r;
                    gate(E::get(o[t * S.so.t]), s, r);
                    go = d * fmaf(a, prev[i], n * xv) * s * r;
                    g = fmaf(d, s, carry);
                }
                gx = n * g;
                gf = g * (prev[i] - xv) * a * n;
                carry = S.reset && S.reset[t * S.B + b] ? 0.f : a * g;
            }
            df[t * S.sdf.t] = E::put(gf); dx[t * S.sdx.t] = E::put(gx);
            if (o) dO[t * S.sdo.t] = E::put(go);
        }
    }
    if (S.dh0) S.dh0[c] = carry;
}

template <int TYPE>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(Scan S, float* __restrict__ h) {
    typedef Elem<TYPE> E; typedef typename E::raw raw;
    const int64_t c = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (c >= S.B * S.H) return;
    const int64_t b = c / S.H; const int j = (int)(c - b * S.H);
    float a, n;
    gate(E::get(((const raw*)S.f)[b * S.sf.b + j]), a, n);
    const float v = n * E::get(((const raw*)S.x)[b * S.sx.b + j]);
    const float s = S.reset && S.reset[b] ? v : fmaf(a, h[c], v);
    h[c] = s;
    ((raw*)S.y)[b * S.sy.b + j] = E::put(S.o ? s * sigmoid(E::get(((const raw*)S.o)[b * S.so.b + j])) : s);
}

// entries (t, b, j) of an output do not fall on each other: either whole steps follow one another or whole sequences do
bool apart(int64_t T, int64_t B, int H, int64_t st, int64_t sb) {
    if (st < 0 || sb < 0) return false;
    if (T <= 1) return B <= 1 || sb >= H;
    if (B <= 1) return st >= H;
    return (sb >= H && st >= (B - 1) * sb + H) || (st >= H && sb >= (T - 1) * st + H);
}
// the last entry's offset stays a 62-bit number
bool reaches(int64_t T, int64_t B, int H, int64_t st, int64_t sb) {
    const __int128 last = (__int128)(T > 0 ? T - 1 : 0) * st + (__int128)(B > 0 ? B - 1 : 0) * sb + H;
    return st >= 0 && sb >= 0 && last < ((__int128)1 << 60);
}
#define APX_SCAN_IN(p, s) APX_REQUIRE(a->p && reaches(a->T, a->B, a->H, a->s##_t, a->s##_b), "input pointer / strides")
#define APX_SCAN_OUT(p, s) APX_REQUIRE(a->p && reaches(a->T, a->B, a->H, a->s##_t, a->s##_b) && apart(a->T, a->B, a->H, a->s##_t, a->s##_b), "output pointer / strides")

int check_common(const apx_gated_scan_args* a) {
    APX_REQUIRE(a, "args");
    APX_REQUIRE(a->type == APX_F32 || a->type == APX_BF16 || a->type == APX_F16, "type");
    APX_REQUIRE(a->T >= 0 && a->B >= 0 && a->H >= 0, "T, B, H");
    APX_REQUIRE((__int128)a->B * a->H < ((__int128)1 << 36), "B * H");
    APX_REQUIRE((__int128)a->B * a->H * (a->T + 1) < ((__int128)1 << 59), "T * B * H");
    return APX_OK;
}
Scan scan_of(const apx_gated_scan_args* a) {
    Scan S = {};
    S.T = a->T; S.B = a->B; S.H = a->H;
    S.f = a->f; S.x = a->x; S.o = a->o; S.dy = a->dy; S.y = a->y; S.df = a->df; S.dx = a->dx; S.do_ = a->do_;
    S.sf = {a->f_t, a->f_b}; S.sx = {a->x_t, a->x_b}; S.so = {a->o_t, a->o_b}; S.sy = {a->y_t, a->y_b};
    S.sdy = {a->dy_t, a->dy_b}; S.sdf = {a->df_t, a->df_b}; S.sdx = {a->dx_t, a->dx_b}; S.sdo = {a->do_t, a->do_b};
    S.h0 = a->h0; S.dh_last = a->dh_last; S.h_last = a->h_last; S.save = a->save; S.dh0 = a->dh0;
    S.reset = a->reset; S.lens = a->lens;
    return S;
}

}  // namespace

#define APX_BY_TYPE(type, kernel, grid, block, s, ...)                                                                    \
    do {                                                                                                                  \
        if ((type) == APX_F32) hipLaunchKernelGGL(kernel<APX_F32>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);           \
        else if ((type) == APX_BF16) hipLaunchKernelGGL(kernel<APX_BF16>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);    \
        else hipLaunchKernelGGL(kernel<APX_F16>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);                             \
        APX_LAUNCH_CHECK();                                                                                               \
    } while (0)

extern "C" size_t apx_gated_scan_save_floats(int64_t T, int64_t B, int H) {
    return T > 0 && B > 0 && H > 0 ? (size_t)((T + KEEP - 1) / KEEP) * (size_t)B * (size_t)H : 0;
}
extern "C" size_t apx_gated_scan_workspace_bytes(int64_t T, int64_t B, int H) { return 0; }

extern "C" int apx_gated_scan_forward(const apx_gated_scan_args* a, void* stream) {
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(a->h_last && a->h_last != a->h0, "h_last is given and is not h0");
    if (a->T > 0) {
        APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_OUT(y, y);
        if (a->o) APX_SCAN_IN(o, o);
        APX_REQUIRE(a->y != a->f && a->y != a->x && a->y != a->o, "y must not lie on an input");
    }
    const Scan S = scan_of(a);
    APX_BY_TYPE(a->type, gated_scan_fwd_kernel, apx_cdiv(a->B * a->H, 64), 64, (hipStream_t)stream, S);
    return APX_OK;
}

extern "C" int apx_gated_scan_backward(const apx_gated_scan_args* a, void* stream) {
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    if (a->T > 0) {
        APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_IN(dy, dy); APX_SCAN_OUT(df, df); APX_SCAN_OUT(dx, dx);
        if (a->o) { APX_SCAN_IN(o, o); APX_SCAN_OUT(do_, do); }
        APX_REQUIRE(a->save, "save of the forward call");
        const void *in[4] = {a->f, a->x, a->dy, a->o}, *out[3] = {a->df, a->dx, a->o ? a->do_ : nullptr};
        for (int i = 0; i < 3; ++i) {
            for (int k = 0; k < 4; ++k) APX_REQUIRE(!out[i] || out[i] != in[k], "an output must not lie on an input");
            for (int k = 0; k < i; ++k) APX_REQUIRE(!out[i] || out[i] != out[k], "outputs must not lie on each other");
        }
    }
    APX_REQUIRE(!a->dh0 || a->dh0 != a->dh_last, "dh0 is not dh_last");
    if (a->T == 0 && !a->dh0) return APX_OK;
    const Scan S = scan_of(a);
    APX_BY_TYPE(a->type, gated_scan_bwd_kernel, apx_cdiv(a->B * a->H, 64), 64, (hipStream_t)stream, S);
    return APX_OK;
}

extern "C" int apx_gated_scan_step(const apx_gated_scan_args* a, float* h, void* stream) {
    APX_REQUIRE(a, "args");
    apx_gated_scan_args one = *a;
    one.T = 1; one.f_t = one.x_t = one.o_t = one.y_t = 0;
    a = &one;
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(h, "h");
    APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_OUT(y, y);
    if (a->o) APX_SCAN_IN(o, o);
    APX_REQUIRE(a->y != a->f && a->y != a->x && a->y != a->o && a->y != (const void*)h, "y must not lie on an input or on h");
    const Scan S = scan_of(a);
    APX_BY_TYPE(a->type, gated_scan_step_kernel, apx_cdiv(a->B * a->H, 256), 256, (hipStream_t)stream, S, h);
    return APX_OK;
}
