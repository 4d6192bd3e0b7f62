// A gated linear recurrence over time-major sequences [T, B, H], its backward pass and its one-step form (include/apx.h, apx_gated_scan_*).
//
//   a = sigmoid(f), n = 1 - a;   p_t = reset ? 0 : h_{t-1};   h_t = a_t p_t + n_t x_t;   y_t = h_t sigmoid(o_t)
//   backward, c_{T-1} = dh_last:  g_t = dy_t sigmoid(o_t) + c_t;   c_{t-1} = reset ? 0 : a_t g_t;   dh0 = c_{-1}
//     dx_t = n_t g_t     df_t = g_t (p_t - x_t) a_t n_t     do_t = dy_t h_t s (1 - s), s = sigmoid(o_t)
//
// The channels (b, j) are independent of each other.  The backward pass needs every h_t again: the forward pass keeps the state in front of every 32nd step (f32), and the steps
// between are run again from there.
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

constexpr int STEPS = 8;                  // steps of a wave in a tile: they stay in its registers
constexpr int WAVES = 8;                  // waves of a workgroup at most
constexpr int KEEP = 32;                  // steps between two kept states; what a tile or a segment begins with is one of them
constexpr int SEGMENTS = 256;             // parts of the time axis at most
constexpr int FILL = 512;                 // workgroups that fill the chip: two for each CU
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

// A run of steps is the map h -> P h + Q.  A reset inside it is P = -0: no product of gates is, products with gates keep it, and it lets nothing of h through (0 times an
// infinity or a NaN would).
__device__ __forceinline__ bool cut(float P) { return __float_as_uint(P) == 0x80000000u; }
template <bool MASK> __device__ __forceinline__ float through(float P, float Q, float h) { return MASK && cut(P) ? Q : fmaf(P, h, Q); }

struct alignas(8) Map { float P, Q; };
struct Strides { int64_t t, b; };
struct Scan {
    int64_t T, B; int H;
    const void *f, *x, *o, *dy; void *y, *df, *dx, *do_;
    Strides sf, sx, so, sy, sdy, sdf, sdx, sdo;
    const float *h0, *dh_last; float *h_last, *save, *dh0;
    const uint8_t* reset; const int32_t* lens;
    int64_t segment; int segments;         // steps of a part of the time axis (a multiple of KEEP), and how many parts
    Map* maps;                          // [segments][B H] the parts' maps
};

template <int TYPE, int VEC> struct Row {
    typedef typename Elem<TYPE>::raw raw;
    struct alignas(VEC * sizeof(raw)) Pack { raw v[VEC]; };
    static __device__ __forceinline__ Pack load(const void* base, int64_t at) { return *(const Pack*)((const raw*)base + at); }
    static __device__ __forceinline__ float get(const Pack& p, int v) { return Elem<TYPE>::get(p.v[v]); }
    static __device__ __forceinline__ void store(void* base, int64_t at, const float (&x)[VEC]) {
        Pack p;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.v[v] = Elem<TYPE>::put(x[v]);
        *(Pack*)((raw*)base + at) = p;
    }
};

// the VEC channels of a lane; beyond the last channel a lane reads the first ones and writes nothing
template <int VEC> struct Channels {
    int64_t c, b; int j; bool on; int64_t len;
    __device__ __forceinline__ Channels(const Scan& S, int group) {
        c = ((int64_t)group * 64 + (threadIdx.x & 63)) * VEC;
        on = c < S.B * S.H;
        if (!on) c = 0;
        b = c / S.H; j = (int)(c - b * S.H);
        len = S.lens ? (int64_t)S.lens[b] : S.T;
    }
};

// a, n of one step of a lane's channels as the maps need them: keep = -0 at a reset, 1 and n = 0 where the step does not count
template <bool MASK> __device__ __forceinline__ void step_gate(float f, bool counts, bool reset, float& a, float& keep, float& n) {
    gate(f, a, n);
    keep = MASK && reset ? -0.f : a;
    if (!counts) { keep = a = 1.f; n = 0.f; }
}

// ------------------------------------------------------------------------------------------------ the maps of the parts (only where the time axis is split)
// forward: h behind the part from h in front of it; BACK: c in front of it from c behind it.  A wave takes a contiguous share of the part.
template <int TYPE, int VEC, bool GATE, bool MASK, bool BACK>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_maps_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    __shared__ Map L[WAVES][64 * VEC];
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    const int64_t share = (S.segment / nw + STEPS - 1) / STEPS * STEPS;
    const int64_t t0 = begin + w * share, t1 = t0 + share < end ? t0 + share : end;
    float P[VEC], Q[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { P[v] = 1.f; Q[v] = 0.f; }
    for (int64_t k = 0; k < share && t0 < end; k += STEPS) {
        typename R::Pack f[STEPS], q[STEPS], o[GATE ? STEPS : 1];
        bool rs[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int64_t u = BACK ? t1 - 1 - k - i : t0 + k + i;
            const int64_t t = u < t0 ? t0 : u < t1 ? u : t1 - 1;
            f[i] = R::load(S.f, t * S.sf.t + ch.b * S.sf.b + ch.j);
            q[i] = BACK ? R::load(S.dy, t * S.sdy.t + ch.b * S.sdy.b + ch.j) : R::load(S.x, t * S.sx.t + ch.b * S.sx.b + ch.j);
            if (GATE) o[i] = R::load(S.o, t * S.so.t + ch.b * S.so.b + ch.j);
            rs[i] = MASK && S.reset && S.reset[t * S.B + ch.b];
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int64_t u = BACK ? t1 - 1 - k - i : t0 + k + i;
            const bool counts = u >= t0 && u < t1 && (!MASK || u < ch.len);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, keep, n;
                step_gate<MASK>(R::get(f[i], v), counts, rs[i], a, keep, n);
                if (BACK) {      // c -> keep (d + c)
                    const float d = GATE ? R::get(q[i], v) * sigmoid(R::get(o[i], v)) : R::get(q[i], v);
                    const float s = counts ? d + Q[v] : Q[v];
                    Q[v] = MASK && cut(keep) ? 0.f : keep * s;
                } else {
                    const float b = counts ? n * R::get(q[i], v) : 0.f;
                    Q[v] = through<MASK>(keep, b, Q[v]);
                }
                P[v] = MASK && cut(keep) ? keep : P[v] * keep;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) L[w][lane * VEC + v] = Map{P[v], Q[v]};
    __syncthreads();
    if (w == 0 && ch.on) {
        Map* out = S.maps + (int64_t)blockIdx.y * S.B * S.H + ch.c;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float p = 1.f, q = 0.f;
            for (int i = 0; i < nw; ++i) {
                const Map m = L[BACK ? nw - 1 - i : i][lane * VEC + v];
                q = through<MASK>(m.P, m.Q, q);
                p = MASK && cut(m.P) ? m.P : p * m.P;
            }
            out[v] = Map{p, q};
        }
    }
}

// what enters a part: `h` carried through the maps of the parts [0, part) - or, BACK, (part, segments) from the last -, a contiguous share of them in each wave
template <int VEC, bool MASK, bool BACK>
__device__ __forceinline__ void enter(const Scan& S, const Channels<VEC>& ch, int part, int w, int nw, Map* L, float (&h)[VEC]) {
    const int lane = threadIdx.x & 63, count = BACK ? S.segments - 1 - part : part;
    if (count == 0) return;
    const int share = (count + nw - 1) / nw, i0 = w * share, i1 = i0 + share < count ? i0 + share : count;
    float P[VEC], Q[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { P[v] = 1.f; Q[v] = 0.f; }
    for (int i = i0; i < i1; ++i) {
        const Map* m = S.maps + (int64_t)(BACK ? S.segments - 1 - i : i) * S.B * S.H + ch.c;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Map q = m[v];
            Q[v] = through<MASK>(q.P, q.Q, Q[v]);
            P[v] = MASK && cut(q.P) ? q.P : P[v] * q.P;
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) L[w * 64 * VEC + lane * VEC + v] = Map{P[v], Q[v]};
    __syncthreads();
    for (int i = 0; i < nw; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Map m = L[i * 64 * VEC + lane * VEC + v];
            h[v] = through<MASK>(m.P, m.Q, h[v]);
        }
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------ forward
// A workgroup walks a part of the time axis of 64 VEC channels in tiles of nw x STEPS steps.  A wave holds its STEPS steps of a tile in registers, the maps of the waves' steps
// meet in LDS (one barrier a tile, two buffers in turn), each wave then runs its own steps again from the state that enters them: one read of the inputs, no step of the chain
// longer than STEPS + nw multiply-adds.
template <int TYPE, int VEC, bool GATE, bool MASK>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_fwd_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    __shared__ Map L[2][WAVES][64 * VEC];
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = S.h0 ? S.h0[ch.c + v] : 0.f;
    enter<VEC, MASK, false>(S, ch, blockIdx.y, w, nw, &L[0][0][0], h);
    int turn = 0;
    for (int64_t tile = begin; tile < end; tile += nw * STEPS, turn ^= 1) {
        const int64_t t0 = tile + w * STEPS;
        float a[STEPS][VEC], b[STEPS][VEC], s[GATE ? STEPS : 1][VEC], P[VEC], Q[VEC];
        {
            typename R::Pack f[STEPS], x[STEPS], o[GATE ? STEPS : 1];
            bool rs[STEPS];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int64_t t = t0 + i < end ? t0 + i : end - 1;
                f[i] = R::load(S.f, t * S.sf.t + ch.b * S.sf.b + ch.j);
                x[i] = R::load(S.x, t * S.sx.t + ch.b * S.sx.b + ch.j);
                if (GATE) o[i] = R::load(S.o, t * S.so.t + ch.b * S.so.b + ch.j);
                rs[i] = MASK && S.reset && S.reset[t * S.B + ch.b];
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) { P[v] = 1.f; Q[v] = 0.f; }
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const bool counts = t0 + i < end && (!MASK || t0 + i < ch.len);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float g, n;
                    step_gate<MASK>(R::get(f[i], v), counts, rs[i], g, a[i][v], n);
                    b[i][v] = counts ? n * R::get(x[i], v) : 0.f;
                    Q[v] = through<MASK>(a[i][v], b[i][v], Q[v]);
                    P[v] = MASK && cut(a[i][v]) ? a[i][v] : P[v] * a[i][v];
                    if (GATE) s[i][v] = sigmoid(R::get(o[i], v));
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) L[turn][w][lane * VEC + v] = Map{P[v], Q[v]};
        __syncthreads();
        float in[VEC];
        for (int i = 0; i < nw; ++i) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (i == w) in[v] = h[v];
                const Map m = L[turn][i][lane * VEC + v];
                h[v] = through<MASK>(m.P, m.Q, h[v]);
            }
        }
        if (!ch.on) continue;
        if (S.save && t0 < end && t0 % KEEP == 0) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) S.save[(t0 / KEEP) * S.B * S.H + ch.c + v] = in[v];
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (t0 + i >= end) break;
            float y[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                in[v] = through<MASK>(a[i][v], b[i][v], in[v]);
                y[v] = GATE ? in[v] * s[i][v] : in[v];
                if (MASK && t0 + i >= ch.len) y[v] = 0.f;
            }
            R::store(S.y, (t0 + i) * S.sy.t + ch.b * S.sy.b + ch.j, y);
        }
    }
    if (w == 0 && ch.on && blockIdx.y == S.segments - 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) S.h_last[ch.c + v] = h[v];
    }
}

// ------------------------------------------------------------------------------------------------ backward
// The same walk from the end.  A tile begins with a kept state; the waves' maps of h (forward in time) and of c (backward: the same product of gates) meet in LDS together.  A wave
// then runs its steps forward for the states and backward for the gradients, on registers alone.
template <int TYPE, int VEC, bool GATE, bool MASK>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_bwd_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    __shared__ float L[2][WAVES][3][64 * VEC];
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    float c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = S.dh_last ? S.dh_last[ch.c + v] : 0.f;
    enter<VEC, MASK, true>(S, ch, blockIdx.y, w, nw, (Map*)&L[0][0][0][0], c);
    int turn = 0;
    const int64_t step = nw * STEPS;
    for (int64_t tile = begin + (end - begin - 1) / step * step; tile >= begin && end > begin; tile -= step, turn ^= 1) {
        const int64_t t0 = tile + w * STEPS;
        // of each step: the gate and 1 minus it, x - later (p - x) a n -, the gradient d of the state's own output; of the output gate the smaller of
        // it and 1 minus it (their product is its derivative, formed without cancellation)
        float a[STEPS][VEC], n[STEPS][VEC], x[STEPS][VEC], d[STEPS][VEC], s[GATE ? STEPS : 1][VEC], dy[GATE ? STEPS : 1][VEC], h[VEC];
        unsigned resets = 0;
        {
            typename R::Pack rf[STEPS], rx[STEPS], rd[STEPS], ro[GATE ? STEPS : 1];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int64_t t = t0 + i < end ? t0 + i : end - 1;
                rf[i] = R::load(S.f, t * S.sf.t + ch.b * S.sf.b + ch.j);
                rx[i] = R::load(S.x, t * S.sx.t + ch.b * S.sx.b + ch.j);
                rd[i] = R::load(S.dy, t * S.sdy.t + ch.b * S.sdy.b + ch.j);
                if (GATE) ro[i] = R::load(S.o, t * S.so.t + ch.b * S.so.b + ch.j);
                if (MASK && S.reset) resets |= (S.reset[t * S.B + ch.b] && t0 + i < end && t0 + i < ch.len ? 1u : 0u) << i;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = S.save[(tile / KEEP) * S.B * S.H + ch.c + v];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const bool counts = t0 + i < end && (!MASK || t0 + i < ch.len);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    gate(R::get(rf[i], v), a[i][v], n[i][v]);
                    if (!counts) { a[i][v] = 1.f; n[i][v] = 0.f; }
                    x[i][v] = counts ? R::get(rx[i], v) : 0.f;
                    const float y = counts ? R::get(rd[i], v) : 0.f;
                    if (GATE) {
                        float g, r;
                        gate(R::get(ro[i], v), g, r);
                        s[i][v] = g < r ? g : r;
                        dy[i][v] = y; d[i][v] = counts ? y * g : 0.f;
                    } else d[i][v] = y;
                }
            }
        }
        auto reset = [&](int i) { return MASK && (resets >> i & 1u); };
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float P = 1.f, Q = 0.f, B = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const float b = n[i][v] * x[i][v];
                Q = reset(i) ? b : fmaf(a[i][v], Q, b);
                P = reset(i) ? -0.f : P * a[i][v];
            }
#pragma unroll
            for (int i = STEPS - 1; i >= 0; --i) B = reset(i) ? 0.f : a[i][v] * (d[i][v] + B);
            L[turn][w][0][lane * VEC + v] = P; L[turn][w][1][lane * VEC + v] = Q; L[turn][w][2][lane * VEC + v] = B;
        }
        __syncthreads();
        float cin[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            for (int i = 0; i < w; ++i) h[v] = through<MASK>(L[turn][i][0][lane * VEC + v], L[turn][i][1][lane * VEC + v], h[v]);
            for (int i = nw - 1; i >= 0; --i) {
                if (i == w) cin[v] = c[v];
                c[v] = through<MASK>(L[turn][i][0][lane * VEC + v], L[turn][i][2][lane * VEC + v], c[v]);
            }
        }
        if (!ch.on) continue;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (t0 + i >= end) break;
            float out[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float p = reset(i) ? 0.f : h[v];
                h[v] = fmaf(a[i][v], p, n[i][v] * x[i][v]);
                x[i][v] = (p - x[i][v]) * a[i][v] * n[i][v];
                if (GATE) {
                    const float r = s[i][v];
                    out[v] = dy[i][v] * h[v] * r * (1.f - r);
                    if (MASK && t0 + i >= ch.len) out[v] = 0.f;
                }
            }
            if (GATE) R::store(S.do_, (t0 + i) * S.sdo.t + ch.b * S.sdo.b + ch.j, out);
        }
#pragma unroll
        for (int i = STEPS - 1; i >= 0; --i) {
            float df[VEC], dx[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float g = d[i][v] + cin[v];
                dx[v] = n[i][v] * g; df[v] = x[i][v] * g;
                if (MASK && t0 + i >= ch.len) dx[v] = df[v] = 0.f;
                cin[v] = reset(i) ? 0.f : a[i][v] * g;
            }
            if (t0 + i < end) {
                R::store(S.df, (t0 + i) * S.sdf.t + ch.b * S.sdf.b + ch.j, df);
                R::store(S.dx, (t0 + i) * S.sdx.t + ch.b * S.sdx.b + ch.j, dx);
            }
        }
    }
    if (w == 0 && ch.on && blockIdx.y == 0 && S.dh0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) S.dh0[ch.c + v] = c[v];
    }
}

// ------------------------------------------------------------------------------------------------ one step
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
#define APX_SCAN_WORKSPACE()                                                                                              \
    do {                                                                                                                  \
        const size_t need = apx_gated_scan_workspace_bytes(a->T, a->B, a->H);                                             \
        APX_REQUIRE(need == 0 || (a->workspace && ((uintptr_t)a->workspace & 15) == 0 && a->workspace_bytes >= need), "workspace"); \
    } while (0)

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

// ------------------------------------------------------------------------------------------------ launches
// How the time axis is split: where the channels alone do not fill the chip, into parts of at least two tiles' steps (a part costs a second look at f and x, and each part folds the
// maps of the parts before it).
struct Split { int64_t groups, segment; int segments; };
Split split(int64_t T, int64_t BH, int vec) {
    Split p;
    p.groups = (BH + 64 * vec - 1) / (64 * vec);
    int64_t want = p.groups >= FILL / 2 ? 1 : FILL / p.groups;
    const int64_t most = T / (WAVES * STEPS);
    if (want > most) want = most;
    if (want > SEGMENTS) want = SEGMENTS;
    if (want < 2) { p.segment = (T + KEEP - 1) / KEEP * KEEP; if (p.segment == 0) p.segment = KEEP; p.segments = 1; return p; }
    p.segment = ((T + want - 1) / want + KEEP - 1) / KEEP * KEEP;
    p.segments = (int)((T + p.segment - 1) / p.segment);
    return p;
}
// waves of a workgroup: a tile of all of them if there are so many steps
int waves(int64_t steps) { return steps >= WAVES * STEPS ? WAVES : steps <= STEPS ? 1 : (int)((steps + STEPS - 1) / STEPS); }

bool aligned(const void* p, int64_t st, int64_t sb, int vec, int bytes) {
    return !p || (((uintptr_t)p % (vec * bytes)) == 0 && st % vec == 0 && sb % vec == 0);
}
template <int TYPE, int VEC, bool GATE, bool MASK> int launch(Scan S, bool back, hipStream_t s) {
    const Split p = split(S.T, S.B * S.H, VEC);
    S.segment = p.segment; S.segments = p.segments;
    const dim3 grid((unsigned)p.groups, p.segments);
    const int nw = waves(S.T < p.segment ? S.T : p.segment);
    if (p.segments > 1) {
        if (back) hipLaunchKernelGGL((gated_scan_maps_kernel<TYPE, VEC, GATE, MASK, true>), grid, dim3(64 * nw), 0, s, S);
        else hipLaunchKernelGGL((gated_scan_maps_kernel<TYPE, VEC, false, MASK, false>), grid, dim3(64 * nw), 0, s, S);
        APX_LAUNCH_CHECK();
    }
    if (back) hipLaunchKernelGGL((gated_scan_bwd_kernel<TYPE, VEC, GATE, MASK>), grid, dim3(64 * nw), 0, s, S);
    else hipLaunchKernelGGL((gated_scan_fwd_kernel<TYPE, VEC, GATE, MASK>), grid, dim3(64 * nw), 0, s, S);
    APX_LAUNCH_CHECK();
    return APX_OK;
}
template <int TYPE, int VEC> int by_masks(const Scan& S, bool back, hipStream_t s) {
    const bool gate = S.o != nullptr, mask = S.reset || S.lens;
    if (gate) return mask ? launch<TYPE, VEC, true, true>(S, back, s) : launch<TYPE, VEC, true, false>(S, back, s);
    return mask ? launch<TYPE, VEC, false, true>(S, back, s) : launch<TYPE, VEC, false, false>(S, back, s);
}
int run(int type, Scan& S, bool back, void* workspace, hipStream_t s) {
    S.maps = (Map*)workspace;
    const int bytes = type == APX_F32 ? 4 : 2;
    bool wide = S.H % 2 == 0;
    const void* p[7] = {S.f, S.x, S.o, back ? S.dy : S.y, back ? S.df : nullptr, back ? S.dx : nullptr, back && S.o ? S.do_ : nullptr};
    const Strides* st[7] = {&S.sf, &S.sx, &S.so, back ? &S.sdy : &S.sy, &S.sdf, &S.sdx, &S.sdo};
    for (int i = 0; i < 7; ++i) wide = wide && aligned(p[i], st[i]->t, st[i]->b, 2, bytes);
    if (type == APX_F32) return wide ? by_masks<APX_F32, 2>(S, back, s) : by_masks<APX_F32, 1>(S, back, s);
    if (type == APX_BF16) return wide ? by_masks<APX_BF16, 2>(S, back, s) : by_masks<APX_BF16, 1>(S, back, s);
    return wide ? by_masks<APX_F16, 2>(S, back, s) : by_masks<APX_F16, 1>(S, back, s);
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
extern "C" size_t apx_gated_scan_workspace_bytes(int64_t T, int64_t B, int H) {
    if (T <= 0 || B <= 0 || H <= 0) return 0;
    size_t most = 0;
    for (int vec = 1; vec <= 2; ++vec) {
        const Split p = split(T, B * H, vec);
        const size_t need = p.segments > 1 ? (size_t)p.segments * B * H * sizeof(Map) : 0;
        if (need > most) most = need;
    }
    return most;
}

extern "C" int apx_gated_scan_forward(const apx_gated_scan_args* a, void* stream) {
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(a->h_last && a->h_last != a->h0, "h_last is given and is not h0");
    if (a->T > 0) {
        APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_OUT(y, y);
        if (a->o) APX_SCAN_IN(o, o);
        APX_REQUIRE(a->y != a->f && a->y != a->x && a->y != a->o, "y must not lie on an input");
    }
    Scan S = scan_of(a);
    APX_SCAN_WORKSPACE();
    return run(a->type, S, false, a->workspace, (hipStream_t)stream);
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
    Scan S = scan_of(a);
    APX_SCAN_WORKSPACE();
    return run(a->type, S, true, a->workspace, (hipStream_t)stream);
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
