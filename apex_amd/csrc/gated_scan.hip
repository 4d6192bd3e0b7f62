// A gated linear recurrence over time-major sequences [T, B, H], its backward pass and its one-step form (include/apx.h, apx_gated_scan_*).
//
//   a = sigmoid(f), n = 1 - a;   p_t = reset ? 0 : h_{t-1};   h_t = a_t p_t + n_t x_t;   y_t = h_t sigmoid(o_t)
//   backward, c_{T-1} = dh_last:  g_t = dy_t sigmoid(o_t) + c_t;   c_{t-1} = reset ? 0 : a_t g_t;   dh0 = c_{-1}
//     dx_t = n_t g_t     df_t = g_t (p_t - x_t) a_t n_t     do_t = dy_t h_t s (1 - s), s = sigmoid(o_t)
//
// The channels (b, j) are independent of each other.  The backward pass needs every h_t again: the forward pass keeps the state in front of every 32nd step (f32, 1/32 of the
// states), and the steps between are run again from there.
//
// What bounds it: memory.  Forward f, x (o) in, y out; backward f, x, dy (o) in, df, dx (do) out: 3 to 7 elements moved for some 45 to 90 vector instructions, so f32 runs at the
// rate of a copy (5.0 TB/s on this card) and 16-bit types are near the rate at which the vector units issue.  Measured on an MI355X, kernel times
// (medians of 23 launches):
//   forward  f32  [400, 1024, 128], resets            124 us   5.1 TB/s        bf16 [32, 4096, 256], resets             44 us   4.8 TB/s
//   backward f32  [400, 1024, 128], output gate       321 us   4.6 TB/s        bf16 [32, 4096, 256], resets             80 us   4.4 TB/s
//   f32 with the output gate, forward 182 us; the pair with lengths of 1 .. 400 (half of the rows are padding and are not read): forward 131 us, backward 252 us
//   forward  bf16 [16384, 4, 256], output gate: maps 15 us + scan 27 us; f32 [65536, 1, 128]: maps 15 + 21 us, backward maps 15 + 30.5 us (the split reads f and x or dy twice)
//   f32 [65536, 1, 8] to [65536, 1, 64]: 11 + 16 to 17 us and 11 + 23 to 25 us, where the bytes take 1 to 8 us: lanes are channels, and below 128 of them a wave's others idle
#include "apx_common.h"
#include <gfx950/dynamic_lds.h>
#include <gfx950/half_types.h>
#include <type_traits>

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

// Steps of a wave in a tile: they stay in its registers.  With 4 one or two more waves fit a SIMD, but each does half the work for the same exchange: bf16 [32, 4096, 256] forward 58 us
// against 43, backward 104 against 77, f32 [400, 1024, 128] with an output gate backward 274 against 251.
constexpr int STEPS = 8;
constexpr int WAVES = 8;                  // waves of a workgroup at most
constexpr int KEEP = 32;                  // steps between two kept states; what a tile begins with is one of them
// Channels of a lane: 2 where H is even (no pair lies across two sequences then).  One channel: bf16 [32, 4096, 256] forward 49 us against 45, backward 97 against 80, f32 the same.
// Four need more registers than there are for enough waves: bf16 backward 125 us.
constexpr int VECTOR = 2;
// The time axis is split into parts where there are SPLIT steps and the channels make fewer than FILL / 2 workgroups: f16 [333, 37, 100] took 30 us forward and 55 us backward
// in one part (29 workgroups) and takes 14 and 20 in six.  FILL workgroups are then wanted: 768 or 1024 made bf16 [16384, 4, 256] 10 % slower, 256 made it 15 % slower.
// SEGMENTS parts at most, because each folds the maps of all before it: 512 made the backward pass of f32 [65536, 1, 128] 40 us instead of 31.
constexpr int SPLIT = 128, FILL = 512, SEGMENTS = 256;
constexpr int FOLD = 16;                  // maps of other parts that a wave has on their way at once (4: 4 us of the 21 to 30 us of a long scan's second pass; 32: registers)
constexpr float LOG2E = 1.44269504088896340736f;

// a = sigmoid(f) and n = 1 - a.  Whichever is below 1/2 is formed without cancellation, the other as 1 minus it: the errors of the fast exponential and reciprocal (1 ulp
// each) then hit a near 1 only in proportion to n, and what a long memory loses and what it takes in differ by the rounding of a alone.  f = +-inf gives exactly 1 and 0, a NaN two.
__device__ __forceinline__ void gate(float f, float& a, float& n) {
    const float e = exp2_fast(-fabsf(f) * LOG2E);
    const float lo = e * rcp_fast(1.f + e), hi = 1.f - lo;
    a = f >= 0.f ? hi : lo;
    n = f >= 0.f ? lo : hi;
}
// the output gate: nothing is carried on with it, so its own value is enough (o = -inf: 1 / inf = 0)
__device__ __forceinline__ float sigmoid(float o) { return rcp_fast(1.f + exp2_fast(-o * LOG2E)); }
// ... and with its derivative s (1 - s) = e / (1 + e)^2, the same for o and -o
__device__ __forceinline__ void sigmoid_slope(float o, float& s, float& slope) {
    const float e = exp2_fast(-fabsf(o) * LOG2E), hi = rcp_fast(1.f + e), lo = e * hi;
    s = o >= 0.f ? hi : lo; slope = lo * hi;
}

// A run of steps is the map h -> P h + Q.  A reset inside it is P = -0: no product of gates is, products with gates keep it, and it lets nothing of h through (0 times an
// infinity or a NaN would).
__device__ __forceinline__ bool cut(float P) { return __float_as_uint(P) == 0x80000000u; }
struct alignas(8) Map { float P, Q; };
template <bool MASK = true> __device__ __forceinline__ float through(const Map& m, float h) { return MASK && cut(m.P) ? m.Q : fmaf(m.P, h, m.Q); }
template <bool MASK = true> __device__ __forceinline__ Map then(const Map& m, const Map& n) {      // m first
    return Map{MASK && cut(n.P) ? n.P : m.P * n.P, through<MASK>(n, m.Q)};
}
struct Strides { int64_t t, b; };         // in bytes
struct Scan {
    int64_t T, B; int H;
    const void *f, *x, *o, *dy; void *y, *df, *dx, *do_;
    Strides sf, sx, so, sy, sdy, sdf, sdx, sdo;
    const float *h0, *dh_last; float *h_last, *save, *dh0;
    const uint8_t* reset; const int32_t* lens;
    bool masked;                           // there are resets or lengths
    int64_t segment; int segments;         // steps of a part of the time axis (a multiple of KEEP), and how many parts
    Map* maps;                             // [segments][B H] the parts' maps
};

template <int TYPE, int VEC> struct Row {
    typedef typename Elem<TYPE>::raw raw;
    typedef raw Pack __attribute__((ext_vector_type(VEC), aligned(sizeof(raw))));      // (one wide access on any boundary that the type allows)
    static __device__ __forceinline__ float get(const Pack& p, int v) { return Elem<TYPE>::get(p[v]); }
    static __device__ __forceinline__ Pack load(const APX_GLOBAL char* wave, unsigned lane) { return *(const APX_GLOBAL Pack*)(wave + lane); }
    static __device__ __forceinline__ void store(APX_GLOBAL char* wave, unsigned lane, const float (&x)[VEC]) {
        Pack p;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = Elem<TYPE>::put(x[v]);
        *(APX_GLOBAL Pack*)(wave + lane) = p;
    }
};

// the VEC channels of a lane, from the first channel of its wave on; beyond the last channel a lane reads what the first lane reads and writes nothing
template <int VEC> struct Channels {
    int64_t c, b0, len, reach; unsigned db, j; bool on;      // reach: where the longest of the wave's sequences ends (nothing behind it is read)
    __device__ __forceinline__ Channels(const Scan& S, int group) {
        const int64_t c0 = (int64_t)group * 64 * VEC;
        c = c0 + (threadIdx.x & 63) * VEC;
        on = c < S.B * S.H;
        if (!on) c = c0;
        b0 = c0 >> 32 ? c0 / S.H : (int64_t)((unsigned)c0 / (unsigned)S.H);      // (a 64-bit division is 100 instructions)
        const unsigned in = (unsigned)(c0 - b0 * S.H) + (unsigned)(c - c0);      // channels from b0's first one on
        db = in / (unsigned)S.H; j = in - db * (unsigned)S.H;
        len = reach = S.T;
        if (S.lens) {
            const int n = S.lens[b0 + db];
            len = n < S.T ? n : S.T;
            int most = n;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) { const int y = __shfl_xor(most, o, 64); most = most > y ? most : y; }
            most = wave_uniform(most);
            reach = most < S.T ? most : S.T;
        }
    }
};
// Where an operand's rows lie: an access is a wave's address of the first of its steps (scalar registers) and 32 bits of a lane's own, one addition further with every step.  (64-bit
// addresses in vector registers took 32 of them and two instructions an access, and one in scalar registers for each access more of those than there are.)
struct Operand {
    char* base; int64_t step; unsigned lane;      // (base as a number: an operand that is not there has none, and is not read)
    template <int VEC> __device__ __forceinline__ Operand(const void* p, const Strides& st, const Channels<VEC>& ch, unsigned bytes)
        : base((char*)((uintptr_t)p + (uintptr_t)(ch.b0 * st.b))), step(st.t), lane(ch.db * (unsigned)st.b + ch.j * bytes) {}
    __device__ __forceinline__ APX_GLOBAL char* at(int64_t t) const { return wave_address(base + t * step); }
    __device__ __forceinline__ unsigned offset(int i) const { return lane_offset(lane + (unsigned)i * (unsigned)step); }
};

// What a step counts for: everything, or - behind a sequence's end, behind the part's - nothing: then a = 1 and n = 0.  Nearly every tile of a wave counts in whole and holds no
// reset; one vote of the wave decides between that form of the arithmetic and the one with the masks (twice the instructions: bf16 [32, 4096, 256] backward 82 us with masks alone).
typedef std::integral_constant<bool, false> Plain;
typedef std::integral_constant<bool, true> Masked;
__device__ __forceinline__ bool nowhere(bool x) { return __builtin_amdgcn_ballot_w64(x) == 0; }

// how many of the STEPS steps from t0 on lie in front of `end`
__device__ __forceinline__ int steps_left(int64_t t0, int64_t end) { return t0 >= end ? 0 : end - t0 < STEPS ? (int)(end - t0) : STEPS; }
// those steps of a lane (at least one; the last one again beyond them)
template <class R> __device__ __forceinline__ void load_steps(typename R::Pack (&q)[STEPS], const Operand& o, int64_t t0, int left) {
    const APX_GLOBAL char* p = o.at(t0);
    unsigned at = o.offset(0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        q[i] = R::load(p, at);
        at += i + 1 < left ? (unsigned)o.step : 0u;
    }
}
__device__ __forceinline__ void load_resets(uint8_t (&r)[STEPS], const Scan& S, const Operand& o, int64_t t0, int left) {
    if (!S.reset) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) r[i] = 0;
        return;
    }
    const APX_GLOBAL char* p = o.at(t0);
    unsigned at = o.offset(0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        r[i] = (uint8_t)p[at];
        at += i + 1 < left ? (unsigned)o.step : 0u;
    }
}
// the steps that are resets, as bits
__device__ __forceinline__ unsigned reset_bits(const uint8_t (&r)[STEPS]) {
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) bits |= (r[i] ? 1u : 0u) << i;
    return bits;
}
// how many of a lane's steps count, and whether in the whole wave all do and none is a reset
template <int VEC> __device__ __forceinline__ bool plain_steps(const Scan& S, const Channels<VEC>& ch, unsigned resets, int64_t t0, int left, int& live) {
    live = left;
    if (S.masked) live = t0 >= ch.len ? 0 : ch.len - t0 < left ? (int)(ch.len - t0) : left;
    return left == STEPS && (!S.masked || nowhere(resets != 0 || live < STEPS));
}

// maps of the waves of a workgroup, two tiles' worth in turn: [2][waves][64 VEC] Map forward, [2][waves][3][64 VEC] floats backward (sized by the launch)
APX_DYNAMIC_LDS(Map, scan_lds, 16);

// ------------------------------------------------------------------------------------------------ a split time axis
// The maps of the parts.  Forward: h behind the part from h in front of it; BACK: c in front of it from c behind it.  A wave takes a contiguous share of the part, STEPS steps at a
// time, the next ones on their way meanwhile.
template <int TYPE, int VEC, bool GATE, bool BACK>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_maps_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    Map* L = scan_lds;
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    const int64_t share = (S.segment / nw + STEPS - 1) / STEPS * STEPS;
    const int64_t stop = end < ch.reach ? end : ch.reach, first = begin + w * share, last = first + share < stop ? first + share : stop;
    const unsigned e = sizeof(typename R::raw);
    const Operand of(S.f, S.sf, ch, e), oq(BACK ? S.dy : S.x, BACK ? S.sdy : S.sx, ch, e), oo(S.o, S.so, ch, e), orst(S.reset, Strides{S.B, 1}, ch, 0);
    Map m[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) m[v] = Map{1.f, 0.f};
    if (first < last) {
        typename R::Pack f[STEPS], q[STEPS], o[GATE ? STEPS : 1];
        uint8_t rs[STEPS];
        auto fetch = [&](int64_t t0) {
            const int left = steps_left(t0, last);
            load_steps<R>(f, of, t0, left);
            load_steps<R>(q, oq, t0, left);
            if constexpr (GATE) load_steps<R>(o, oo, t0, left);
            load_resets(rs, S, orst, t0, left);
            __builtin_amdgcn_sched_barrier(0);
        };
        const int64_t tiles = (last - first + STEPS - 1) / STEPS;
        fetch(first + (BACK ? tiles - 1 : 0) * STEPS);
        for (int64_t k = 0; k < tiles; ++k) {
            const int64_t t0 = first + (BACK ? tiles - 1 - k : k) * STEPS;
            const unsigned resets = reset_bits(rs);
            int live;
            const bool plain = plain_steps(S, ch, resets, t0, steps_left(t0, last), live);
            Map one[STEPS][VEC];
            auto steps = [&](auto masked) {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        float a, n;
                        gate(R::get(f[i], v), a, n);
                        float x = R::get(q[i], v);
                        if constexpr (GATE) x *= sigmoid(R::get(o[i], v));
                        one[i][v] = Map{a, BACK ? a * x : n * x};      // BACK: c -> a (d + c)
                        if (masked) {
                            if (resets >> i & 1u) one[i][v] = Map{-0.f, BACK ? 0.f : one[i][v].Q};
                            if (i >= live) one[i][v] = Map{1.f, 0.f};
                        }
                    }
                }
            };
            if (plain) steps(Plain()); else steps(Masked());
            if (k + 1 < tiles) fetch(first + (BACK ? tiles - 2 - k : k + 1) * STEPS);
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) m[v] = plain ? then<false>(m[v], one[BACK ? STEPS - 1 - i : i][v]) : then(m[v], one[BACK ? STEPS - 1 - i : i][v]);
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) L[(w * 64 + lane) * VEC + v] = m[v];
    __syncthreads();
    if (w == 0 && ch.on) {
        Map* out = S.maps + (int64_t)blockIdx.y * S.B * S.H + ch.c;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            Map all = {1.f, 0.f};
            for (int i = 0; i < nw; ++i) all = then(all, L[((BACK ? nw - 1 - i : i) * 64 + lane) * VEC + v]);
            out[v] = all;
        }
    }
}

// what enters a part: `h` carried through the maps of the parts [0, part) - or, BACK, (part, segments) from the last -, a contiguous share of them in each wave
template <int VEC, bool BACK>
__device__ __forceinline__ void enter(const Scan& S, const Channels<VEC>& ch, int part, int w, int nw, Map* L, float (&h)[VEC]) {
    const int lane = threadIdx.x & 63, count = BACK ? S.segments - 1 - part : part;
    if (count == 0) return;
    const int share = (count + nw - 1) / nw, i0 = w * share, i1 = i0 + share < count ? i0 + share : count;
    Map m[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) m[v] = Map{1.f, 0.f};
    auto batch = [&](int i, auto many) {      // that many maps on their way at once: they are what a workgroup waits for first
        constexpr int N = many;
        Map q[N][VEC];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = i + k < i1 ? i + k : i;
            const Map* p = S.maps + (int64_t)(BACK ? S.segments - 1 - at : at) * S.B * S.H + ch.c;
#pragma unroll
            for (int v = 0; v < VEC; ++v) q[k][v] = p[v];
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) if (i + k < i1) m[v] = then(m[v], q[k][v]);
    };
    if (share > 4) for (int i = i0; i < i1; i += FOLD) batch(i, std::integral_constant<int, FOLD>());
    else if (i0 < i1) batch(i0, std::integral_constant<int, 4>());
#pragma unroll
    for (int v = 0; v < VEC; ++v) L[w * 64 * VEC + lane * VEC + v] = m[v];
    __syncthreads();
    for (int i = 0; i < nw; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = through(L[i * 64 * VEC + lane * VEC + v], h[v]);
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------ forward
// A workgroup walks a part of the time axis of 64 VEC channels in tiles of nw x STEPS steps.  A wave holds its STEPS steps of a tile in registers, the maps of the waves' steps
// meet in LDS (one barrier a tile, two buffers in turn), each wave then runs its own steps again from the state that enters them: one read of the inputs, no step of the chain
// longer than STEPS + nw multiply-adds.  Without an output gate the next tile's loads are issued before this one's barrier (f32 [400, 1024, 128] 158 -> 131 us); with one there are not
// the registers for it (175 -> 190 us).
template <int TYPE, int VEC, bool GATE>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_fwd_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    constexpr bool AHEAD = !GATE;
    Map* L = scan_lds;
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t step = nw * STEPS, begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = S.h0 ? S.h0[ch.c + v] : 0.f;
    const unsigned e = sizeof(typename R::raw);
    const Operand of(S.f, S.sf, ch, e), ox(S.x, S.sx, ch, e), oo(S.o, S.so, ch, e), oy(S.y, S.sy, ch, e), orst(S.reset, Strides{S.B, 1}, ch, 0);
    typename R::Pack f[STEPS], x[STEPS], o[GATE ? STEPS : 1];
    uint8_t rs[STEPS];
    const int64_t stop = end < ch.reach ? end : ch.reach;
    auto fetch = [&](int64_t t0) {
        const int left = steps_left(t0, stop);
        if (left == 0) return;
        load_steps<R>(f, of, t0, left);
        load_steps<R>(x, ox, t0, left);
        if constexpr (GATE) load_steps<R>(o, oo, t0, left);
        load_resets(rs, S, orst, t0, left);
        __builtin_amdgcn_sched_barrier(0);
    };
    int turn = 0;
    if (AHEAD && begin < end) fetch(begin + w * STEPS);
    enter<VEC, false>(S, ch, blockIdx.y, w, nw, L, h);
    for (int64_t tile = begin; tile < end; tile += step, turn ^= 1) {
        const int64_t t0 = tile + w * STEPS;
        if (!AHEAD) fetch(t0);
        Map one[STEPS][VEC], m[VEC];
        const unsigned resets = reset_bits(rs);
        const int left = steps_left(t0, end);
        int live;
        const bool plain = plain_steps(S, ch, resets, t0, left, live);
        const bool none = t0 >= stop;
        if (none) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) m[v] = Map{1.f, 0.f};
        }
        auto maps = [&](auto masked) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    float a, n;
                    gate(R::get(f[i], v), a, n);
                    one[i][v] = Map{a, n * R::get(x[i], v)};
                    if (masked) {
                        if (resets >> i & 1u) one[i][v].P = -0.f;
                        if (i >= live) one[i][v] = Map{1.f, 0.f};
                    }
                    m[v] = i == 0 ? one[i][v] : then<masked>(m[v], one[i][v]);
                }
            }
        };
        if (plain) maps(Plain()); else if (!none) maps(Masked());
        if (AHEAD && tile + step < end) fetch(t0 + step);
#pragma unroll
        for (int v = 0; v < VEC; ++v) L[((turn * nw + w) * 64 + lane) * VEC + v] = m[v];
        __syncthreads();
        float in[VEC];
#pragma unroll 4
        for (int i = 0; i < nw; ++i) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (i == w) in[v] = h[v];
                const Map k = L[((turn * nw + i) * 64 + lane) * VEC + v];
                h[v] = S.masked ? through(k, h[v]) : through<false>(k, h[v]);
            }
        }
        if (!ch.on) continue;
        if (S.save && t0 < end && t0 % KEEP == 0) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) S.save[(t0 / KEEP) * S.B * S.H + ch.c + v] = in[v];
        }
        APX_GLOBAL char* const py = oy.at(t0);
        unsigned at = oy.offset(0);
        auto outputs = [&](auto masked) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i, at += (unsigned)oy.step) {
                if (masked && i >= left) break;
                float y[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    in[v] = through<masked>(one[i][v], in[v]);
                    y[v] = in[v];
                    if constexpr (GATE) y[v] *= sigmoid(R::get(o[i], v));
                    if (masked && i >= live) y[v] = 0.f;
                }
                R::store(py, at, y);
            }
        };
        if (plain) outputs(Plain());
        else if (!none) outputs(Masked());
        else {
            const float zero[VEC] = {};
            for (int i = 0; i < left; ++i, at += (unsigned)oy.step) R::store(py, at, zero);
        }
    }
    if (w == 0 && ch.on && end == S.T) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) S.h_last[ch.c + v] = h[v];
    }
}

// ------------------------------------------------------------------------------------------------ backward
// The same walk from the end.  A tile begins with a kept state; the waves' maps of h (forward in time) and of c (backward: the same product of gates) meet in LDS together.  A wave
// then runs its steps forward for the states and backward for the gradients, on registers alone.  (f32 without an output gate needs 183 of them, with one 229: 2 waves a SIMD,
// enough for the memory.  Held to 128 by the launch bounds the compiler spills: 700 us for 321.  The output gate is evaluated twice rather than kept.)
template <int TYPE, int VEC, bool GATE>
__global__ __launch_bounds__(64 * WAVES) void gated_scan_bwd_kernel(Scan S) {
    typedef Row<TYPE, VEC> R;
    constexpr bool AHEAD = !GATE;
    float* const L = (float*)(Map*)scan_lds;
    const int lane = threadIdx.x & 63, w = wave_uniform(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Channels<VEC> ch(S, blockIdx.x);
    const int64_t step = nw * STEPS, begin = (int64_t)blockIdx.y * S.segment, end = begin + S.segment < S.T ? begin + S.segment : S.T;
    float c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = S.dh_last ? S.dh_last[ch.c + v] : 0.f;
    const unsigned e = sizeof(typename R::raw);
    const Operand of(S.f, S.sf, ch, e), ox(S.x, S.sx, ch, e), ody(S.dy, S.sdy, ch, e), oo(S.o, S.so, ch, e), odf(S.df, S.sdf, ch, e), odx(S.dx, S.sdx, ch, e), odo(S.do_, S.sdo, ch, e),
        orst(S.reset, Strides{S.B, 1}, ch, 0);
    typename R::Pack rf[STEPS], rx[STEPS], rd[STEPS], ro[GATE ? STEPS : 1];
    uint8_t rs[STEPS];
    float kept[VEC];
    const int64_t stop = end < ch.reach ? end : ch.reach;
    auto fetch = [&](int64_t tile) {
        const int64_t t0 = tile + w * STEPS;
        const int left = steps_left(t0, stop);
        if (left == 0) return;
        load_steps<R>(rf, of, t0, left);
        load_steps<R>(rx, ox, t0, left);
        load_steps<R>(rd, ody, t0, left);
        if constexpr (GATE) load_steps<R>(ro, oo, t0, left);
        load_resets(rs, S, orst, t0, left);
#pragma unroll
        for (int v = 0; v < VEC; ++v) kept[v] = S.save[(tile / KEEP) * S.B * S.H + ch.c + v];
        __builtin_amdgcn_sched_barrier(0);
    };
    int turn = 0;
    auto at = [&](int wave, int k) { return L + (((turn * nw + wave) * 3 + k) * 64 + lane) * VEC; };
    const int64_t last = begin + (end - begin - 1) / step * step;
    if (AHEAD && begin < end) fetch(last);
    enter<VEC, true>(S, ch, blockIdx.y, w, nw, scan_lds, c);
    for (int64_t tile = last; tile >= begin && end > begin; tile -= step, turn ^= 1) {
        const int64_t t0 = tile + w * STEPS;
        if (!AHEAD) fetch(tile);
        // of each step: the gate and 1 minus it, x - later (p - x) a n -, and dy - later the gradient of the state's own output, dy sigmoid(o)
        float a[STEPS][VEC], n[STEPS][VEC], x[STEPS][VEC], d[STEPS][VEC], h[VEC];
        const unsigned resets = reset_bits(rs);
        const int left = steps_left(t0, end);
        int live;
        const bool plain = plain_steps(S, ch, resets, t0, left, live);
        const bool none = t0 >= stop;
        if (none) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) { at(w, 0)[v] = 1.f; at(w, 1)[v] = at(w, 2)[v] = h[v] = 0.f; }
        }
        auto maps = [&](auto masked) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float P = 1.f, Q = 0.f, C = 0.f;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const bool counts = !masked || i < live, reset = masked && counts && (resets >> i & 1u);
                    gate(R::get(rf[i], v), a[i][v], n[i][v]);
                    if (!counts) { a[i][v] = 1.f; n[i][v] = 0.f; }
                    x[i][v] = counts ? R::get(rx[i], v) : 0.f;
                    const float y = counts ? R::get(rd[i], v) : 0.f;
                    d[i][v] = y;
                    const float b = n[i][v] * x[i][v];
                    Q = reset ? b : fmaf(a[i][v], Q, b);
                    P *= a[i][v];
                }
                // A reset anywhere in the steps cuts both maps.  Of h, that lies in the order of the steps: a gate behind it that is a NaN is one in Q too.  Of c, a NaN behind it must
                // not come through: the product of gates is not asked.
                if (masked && (resets & ((1u << live) - 1u))) P = -0.f;
#pragma unroll
                for (int i = STEPS - 1; i >= 0; --i) {
                    float g = d[i][v];
                    if constexpr (GATE) { g *= sigmoid(R::get(ro[i], v)); if (masked && i >= live) g = 0.f; }
                    C = masked && (resets >> i & 1u) && i < live ? 0.f : a[i][v] * (g + C);
                }
                at(w, 0)[v] = P; at(w, 1)[v] = Q; at(w, 2)[v] = C;
                h[v] = kept[v];
            }
        };
        if (plain) maps(Plain()); else if (!none) maps(Masked());
        if (AHEAD && tile > begin) fetch(tile - step);
        __syncthreads();
        float cin[VEC];
        auto fold = [&](auto masked) {
#pragma unroll 2
            for (int i = 0; i < w; ++i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) h[v] = through<masked>(Map{at(i, 0)[v], at(i, 1)[v]}, h[v]);
#pragma unroll 2
            for (int i = nw - 1; i >= 0; --i)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    if (i == w) cin[v] = c[v];
                    c[v] = through<masked>(Map{at(i, 0)[v], at(i, 2)[v]}, c[v]);
                }
        };
        if (S.masked) fold(Masked()); else fold(Plain());
        if (!ch.on) continue;
        APX_GLOBAL char *const pdo = odo.at(t0), *const pdf = odf.at(t0), *const pdx = odx.at(t0);
        unsigned ado = odo.offset(0), adf = odf.offset(STEPS - 1), adx = odx.offset(STEPS - 1);
        auto outputs = [&](auto masked) {
            auto counts = [&](int i) { return !masked || i < live; };
            auto reset = [&](int i) { return masked && (resets >> i & 1u) && counts(i); };
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                float out[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float p = reset(i) ? 0.f : h[v];
                    h[v] = fmaf(a[i][v], p, n[i][v] * x[i][v]);
                    x[i][v] = (p - x[i][v]) * (a[i][v] * n[i][v]);
                    if constexpr (GATE) {
                        float g, slope;
                        sigmoid_slope(R::get(ro[i], v), g, slope);
                        out[v] = counts(i) ? d[i][v] * h[v] * slope : 0.f;
                        d[i][v] = counts(i) ? d[i][v] * g : 0.f;
                    }
                }
                if constexpr (GATE) { if (!masked || i < left) R::store(pdo, ado, out); ado += (unsigned)odo.step; }
            }
#pragma unroll
            for (int i = STEPS - 1; i >= 0; --i) {
                float df[VEC], dx[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float g = d[i][v] + cin[v];
                    dx[v] = n[i][v] * g; df[v] = x[i][v] * g;
                    if (!counts(i)) dx[v] = df[v] = 0.f;
                    cin[v] = reset(i) ? 0.f : a[i][v] * g;
                }
                if (!masked || i < left) {
                    R::store(pdf, adf, df);
                    R::store(pdx, adx, dx);
                }
                adf -= (unsigned)odf.step; adx -= (unsigned)odx.step;
            }
        };
        if (plain) outputs(Plain());
        else if (!none) outputs(Masked());
        else {
            const float zero[VEC] = {};
            for (int i = 0; i < left; ++i) {
                R::store(pdf, odf.offset(i), zero);
                R::store(pdx, odx.offset(i), zero);
                if constexpr (GATE) R::store(pdo, odo.offset(i), zero);
            }
        }
    }
    if (w == 0 && ch.on && begin == 0 && S.dh0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) S.dh0[ch.c + v] = c[v];
    }
}

// ------------------------------------------------------------------------------------------------ one step
struct OneStep { const void *f, *x, *o; void* y; int64_t fb, xb, ob, yb; const uint8_t* reset; unsigned channels, H; };      // rows so many bytes apart
template <int TYPE>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(OneStep S, float* __restrict__ h) {
    typedef Elem<TYPE> E; typedef typename E::raw raw;
    const unsigned c = blockIdx.x * 256u + threadIdx.x;
    if (c >= S.channels) return;
    const unsigned b = c / S.H, j = c - b * S.H;
    auto at = [&](const void* p, int64_t row) { return *(const raw*)((const char*)p + b * row + j * sizeof(raw)); };
    float a, n;
    gate(E::get(at(S.f, S.fb)), a, n);
    const float v = n * E::get(at(S.x, S.xb));
    const float s = S.reset && S.reset[b] ? v : fmaf(a, h[c], v);
    h[c] = s;
    *(raw*)((char*)S.y + b * S.yb + j * sizeof(raw)) = E::put(S.o ? s * sigmoid(E::get(at(S.o, S.ob))) : s);
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
// What an operand takes of memory: rows of `row` bytes, n[k] of them s[k] bytes apart along each of two axes (an axis of one row, or of the same row again, has none).
struct Span { uintptr_t at; int64_t n[2], s[2], row; };
Span span(const void* p, int64_t nt, int64_t st, int64_t nb, int64_t sb, int64_t row) {
    Span a = {(uintptr_t)p, {nt, nb}, {st, sb}, row};
    for (int k = 0; k < 2; ++k) if (a.n[k] <= 1 || a.s[k] == 0) { a.n[k] = 1; a.s[k] = 0; }
    return a;
}
Span dense(const void* p, int64_t bytes) { return span(p, 1, 0, 1, 0, bytes); }
uintptr_t behind(const Span& a) { return a.at + (a.n[0] - 1) * a.s[0] + (a.n[1] - 1) * a.s[1] + a.row; }
int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y < 0); }
// Do rows of a and b of the same strides share a byte?  The difference of their beginnings is i S + j s + r with numbers of steps i, j and |r| below a row's length; where S is more than
// all that j s + r can be, and s more than r, two candidates for each are all there are.  -1: the strides are not the same, or not so far apart.
int meets_alike(const Span& a, const Span& b) {
    int64_t s[2];
    for (int k = 0; k < 2; ++k) {
        if (a.n[k] > 1 && b.n[k] > 1 && a.s[k] != b.s[k]) return -1;
        s[k] = a.n[k] > 1 ? a.s[k] : b.s[k];
    }
    const int far = s[0] >= s[1] ? 0 : 1, near = 1 - far;
    const int64_t row = a.row > b.row ? a.row : b.row, n = a.n[near] > b.n[near] ? a.n[near] : b.n[near], D = (int64_t)(b.at - a.at);
    if ((s[near] && s[near] < row) || (s[far] && s[far] < (n - 1) * s[near] + row)) return -1;
    const int64_t i0 = s[far] ? floor_div(D, s[far]) : 0;
    for (int64_t i = i0; i <= i0 + (s[far] != 0); ++i) {
        if (i < 1 - b.n[far] || i > a.n[far] - 1) continue;
        const int64_t rest = D - i * s[far], j0 = s[near] ? floor_div(rest, s[near]) : 0;
        for (int64_t j = j0; j <= j0 + (s[near] != 0); ++j) {
            if (j < 1 - b.n[near] || j > a.n[near] - 1) continue;
            const int64_t r = rest - j * s[near];
            if (-b.row < r && r < a.row) return 1;
        }
    }
    return 0;
}
// rows that lie apart and thus follow one another
bool in_a_row(const Span& a) {
    const int far = a.s[0] >= a.s[1] ? 0 : 1, near = 1 - far;
    return (a.s[near] == 0 || a.s[near] >= a.row) && (a.s[far] == 0 || a.s[far] >= (a.n[near] - 1) * a.s[near] + a.row);
}
// Does an operand whose rows follow one another share a byte with [at, at + bytes)?  The last row that begins at or in front of `at` does, or the next one does.
bool meets_row(const Span& out, uintptr_t at, int64_t bytes) {
    const int far = out.s[0] >= out.s[1] ? 0 : 1, near = 1 - far;
    const int64_t D = (int64_t)(at - out.at);
    if (D < 0) return D + bytes > 0;
    int64_t i = out.s[far] ? D / out.s[far] : 0;
    if (i >= out.n[far]) i = out.n[far] - 1;
    const int64_t rest = D - i * out.s[far];
    int64_t j = out.s[near] ? rest / out.s[near] : 0;
    if (j >= out.n[near]) j = out.n[near] - 1;
    if (rest - j * out.s[near] < out.row) return true;
    if (j + 1 < out.n[near]) return i * out.s[far] + (j + 1) * out.s[near] < D + bytes;
    return i + 1 < out.n[far] && (i + 1) * out.s[far] < D + bytes;
}
// ... with another operand?  Exact where their strides are the same - slices of one buffer - or the other has few rows; else all rows on one pitch that keep to columns of their own are
// apart, and what is left counts as sharing.
bool meets(const Span& out, const Span& b) {
    if (behind(out) <= b.at || behind(b) <= out.at) return false;
    if (b.n[0] == 1 && b.n[1] == 1) return meets_row(out, b.at, b.row);
    if (out.n[0] == 1 && out.n[1] == 1 && in_a_row(b)) return meets_row(b, out.at, out.row);
    const int alike = meets_alike(out, b);
    if (alike >= 0) return alike;
    int64_t pitch = 0;
    for (const Span* a : {&out, &b}) for (int k = 0; k < 2; ++k) for (int64_t y = a->s[k]; y; ) { const int64_t x = pitch; pitch = y; y = x % y; }
    const int64_t D = (int64_t)(b.at - out.at), column = D - floor_div(D, pitch) * pitch;
    if (column >= out.row && column + b.row <= pitch) return false;
    if (b.n[0] > 4096 / b.n[1]) return true;
    for (int64_t i = 0; i < b.n[0]; ++i) for (int64_t j = 0; j < b.n[1]; ++j) if (meets_row(out, b.at + i * b.s[0] + j * b.s[1], b.row)) return true;
    return false;
}
// the operands of a call: outputs first
struct Spans {
    Span a[16]; int n = 0, outputs = 0;
    void add(const Span& s) { a[n++] = s; }
    bool apart() const {
        for (int i = 0; i < outputs; ++i) for (int k = i + 1; k < n; ++k) if (meets(a[i], a[k])) return false;
        return true;
    }
};
bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
size_t size_of(int type) { return type == APX_F32 ? 4 : 2; }
#define APX_SCAN_IN(p, s) APX_REQUIRE(a->p && aligned(a->p, size_of(a->type)) && reaches(a->T, a->B, a->H, a->s##_t, a->s##_b), "input pointer / strides")
#define APX_SCAN_OUT(p, s) APX_REQUIRE(a->p && aligned(a->p, size_of(a->type)) && reaches(a->T, a->B, a->H, a->s##_t, a->s##_b) && apart(a->T, a->B, a->H, a->s##_t, a->s##_b), "output pointer / strides")
#define APX_SCAN_WORKSPACE()                                                                                              \
    do {                                                                                                                  \
        const size_t need = apx_gated_scan_workspace_bytes(a->T, a->B, a->H);                                             \
        APX_REQUIRE(need == 0 || (a->workspace && ((uintptr_t)a->workspace & 15) == 0 && a->workspace_bytes >= need), "workspace");                \
    } while (0)

bool sizes_fit(int64_t T, int64_t B, int H) {
    return T >= 0 && B >= 0 && H >= 0 && T < ((int64_t)1 << 40) && (__int128)B * H < ((__int128)1 << 36) && (__int128)B * H * (T + 1) < ((__int128)1 << 59);
}
int check_common(const apx_gated_scan_args* a) {
    APX_REQUIRE(a, "args");
    APX_REQUIRE(a->type == APX_F32 || a->type == APX_BF16 || a->type == APX_F16, "type");
    APX_REQUIRE(sizes_fit(a->T, a->B, a->H), "T, B, H");
    return APX_OK;
}
// Only what the direction uses is looked at and handed on: a field that is not read may hold anything.
Scan scan_of(const apx_gated_scan_args* a, bool back) {
    Scan S = {};
    S.T = a->T; S.B = a->B; S.H = a->H;
    const int64_t e = size_of(a->type);
    if (a->T > 0) {
        S.f = a->f; S.sf = {a->f_t * e, a->f_b * e};
        S.x = a->x; S.sx = {a->x_t * e, a->x_b * e};
        if (a->o) { S.o = a->o; S.so = {a->o_t * e, a->o_b * e}; }
        if (back) {
            S.dy = a->dy; S.sdy = {a->dy_t * e, a->dy_b * e};
            S.df = a->df; S.sdf = {a->df_t * e, a->df_b * e};
            S.dx = a->dx; S.sdx = {a->dx_t * e, a->dx_b * e};
            if (a->o) { S.do_ = a->do_; S.sdo = {a->do_t * e, a->do_b * e}; }
        } else { S.y = a->y; S.sy = {a->y_t * e, a->y_b * e}; }
        S.reset = a->reset; S.lens = a->lens; S.save = a->save;
    }
    if (back) { S.dh_last = a->dh_last; S.dh0 = a->dh0; }
    else { S.h0 = a->h0; S.h_last = a->h_last; }
    return S;
}

Spans spans_of(const Scan& S, const apx_gated_scan_args* a, bool back) {
    Spans all;
    const int64_t row = S.H * (int64_t)size_of(a->type), state = S.B * S.H * 4;
    auto operand = [&](const void* p, const Strides& st) { if (p) all.add(span(p, S.T, st.t, S.B, st.b, row)); };
    auto flat = [&](const void* p, size_t bytes) { if (p && bytes) all.add(dense(p, (int64_t)bytes)); };
    const size_t save = apx_gated_scan_save_floats(S.T, S.B, S.H) * 4;
    if (back) { operand(S.df, S.sdf); operand(S.dx, S.sdx); operand(S.do_, S.sdo); flat(S.dh0, state); }
    else { operand(S.y, S.sy); flat(S.h_last, state); flat(S.save, save); }
    flat(a->workspace, apx_gated_scan_workspace_bytes(S.T, S.B, S.H));
    all.outputs = all.n;
    operand(S.f, S.sf); operand(S.x, S.sx); operand(S.o, S.so);
    if (back) { operand(S.dy, S.sdy); flat(S.save, save); flat(S.dh_last, state); }
    else flat(S.h0, state);
    flat(S.reset, S.T * S.B); flat(S.lens, S.B * 4);
    return all;
}

// ------------------------------------------------------------------------------------------------ launches
// how the time axis is split: into parts of whole kept stretches
struct Split { int64_t groups, segment; int segments; };
Split split(int64_t T, int64_t BH, int vec) {
    Split p;
    p.groups = (BH + 64 * vec - 1) / (64 * vec);
    int64_t want = T < SPLIT || p.groups >= FILL / 2 ? 1 : FILL / p.groups;
    if (want > T / KEEP) want = T / KEEP;
    if (want > SEGMENTS) want = SEGMENTS;
    if (want < 2) want = 1;
    p.segment = ((T + want - 1) / want + KEEP - 1) / KEEP * KEEP;
    if (p.segment == 0) p.segment = KEEP;
    p.segments = T ? (int)((T + p.segment - 1) / p.segment) : 1;
    return p;
}
// waves of a workgroup: a tile of all of them if there are so many steps (the tiles of a loop then begin at kept states)
int waves(int64_t steps) { return steps >= WAVES * STEPS ? WAVES : steps <= STEPS ? 1 : (int)((steps + STEPS - 1) / STEPS); }

template <int TYPE, int VEC, bool GATE> int launch(Scan S, bool back, hipStream_t s) {
    const Split p = split(S.T, S.B * S.H, VEC);
    S.segment = p.segment; S.segments = p.segments;
    S.masked = S.reset || S.lens;
    // what a wave touches in a tile - STEPS steps of the sequences that its 64 VEC channels belong to - lies within 4 GB; `last`: how many sequences behind its first one
    const int64_t steps = (S.T < STEPS ? S.T : STEPS) - 1, n = 64 * VEC, more = S.H % n == 0 ? 0 : n % S.H == 0 ? n / S.H - 1 : n / S.H + 1, last = S.B - 1 < more ? S.B - 1 : more;
    for (const Strides* st : {&S.sf, &S.sx, &S.so, &S.sy, &S.sdy, &S.sdf, &S.sdx, &S.sdo})
        APX_REQUIRE((S.T <= 1 || st->t < ((int64_t)1 << 32)) && (last == 0 || st->b < ((int64_t)1 << 32)) &&
                    (S.T <= 1 ? 0 : steps * st->t) + last * (last ? st->b : 0) + 4ll * S.H < ((int64_t)1 << 32), "neighbouring steps or sequences lie too far apart");
    APX_REQUIRE((S.T <= 1 ? 0 : steps * S.B) + last < ((int64_t)1 << 32), "B");
    const dim3 grid((unsigned)p.groups, p.segments), block(64 * waves(S.T < p.segment ? S.T : p.segment));
    APX_REQUIRE(p.groups * block.x < ((int64_t)1 << 32), "B * H");
    const size_t maps = block.x * VEC * sizeof(Map);      // LDS for one map a thread and channel
    if (p.segments > 1) {
        if (back) hipLaunchKernelGGL((gated_scan_maps_kernel<TYPE, VEC, GATE, true>), grid, block, maps, s, S);
        else hipLaunchKernelGGL((gated_scan_maps_kernel<TYPE, VEC, false, false>), grid, block, maps, s, S);
        APX_LAUNCH_CHECK();
    }
    if (back) hipLaunchKernelGGL((gated_scan_bwd_kernel<TYPE, VEC, GATE>), grid, block, 3 * maps, s, S);
    else hipLaunchKernelGGL((gated_scan_fwd_kernel<TYPE, VEC, GATE>), grid, block, 2 * maps, s, S);
    APX_LAUNCH_CHECK();
    return APX_OK;
}
template <int TYPE> int by_width(const Scan& S, bool back, hipStream_t s) {
    if (S.H % VECTOR == 0) return S.o ? launch<TYPE, VECTOR, true>(S, back, s) : launch<TYPE, VECTOR, false>(S, back, s);
    return S.o ? launch<TYPE, 1, true>(S, back, s) : launch<TYPE, 1, false>(S, back, s);
}
int run(int type, Scan& S, bool back, void* workspace, hipStream_t s) {
    S.maps = (Map*)workspace;
    return type == APX_F32 ? by_width<APX_F32>(S, back, s) : type == APX_BF16 ? by_width<APX_BF16>(S, back, s) : by_width<APX_F16>(S, back, s);
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
    return T > 0 && B > 0 && H > 0 && sizes_fit(T, B, H) ? (size_t)((T + KEEP - 1) / KEEP) * (size_t)B * (size_t)H : 0;
}
extern "C" size_t apx_gated_scan_workspace_bytes(int64_t T, int64_t B, int H) {
    if (T <= 0 || B <= 0 || H <= 0 || !sizes_fit(T, B, H)) return 0;
    const Split p = split(T, B * H, H % VECTOR == 0 ? VECTOR : 1);
    return p.segments > 1 ? (size_t)p.segments * B * H * sizeof(Map) : 0;
}

extern "C" int apx_gated_scan_forward(const apx_gated_scan_args* a, void* stream) {
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(a->h_last, "h_last");
    APX_REQUIRE(aligned(a->h0, 4) && aligned(a->h_last, 4) && aligned(a->lens, 4) && aligned(a->save, 4), "4-byte alignment");
    if (a->T > 0) {
        APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_OUT(y, y);
        if (a->o) APX_SCAN_IN(o, o);
    }
    Scan S = scan_of(a, false);
    APX_SCAN_WORKSPACE();
    APX_REQUIRE(spans_of(S, a, false).apart(), "an output overlaps an input or another output");
    return run(a->type, S, false, a->workspace, (hipStream_t)stream);
}

extern "C" int apx_gated_scan_backward(const apx_gated_scan_args* a, void* stream) {
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(aligned(a->h0, 4) && aligned(a->dh_last, 4) && aligned(a->dh0, 4) && aligned(a->lens, 4) && aligned(a->save, 4), "4-byte alignment");
    if (a->T > 0) {
        APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_IN(dy, dy); APX_SCAN_OUT(df, df); APX_SCAN_OUT(dx, dx);
        if (a->o) { APX_SCAN_IN(o, o); APX_SCAN_OUT(do_, do); }
        APX_REQUIRE(a->save, "save of the forward call");
    }
    if (a->T == 0 && !a->dh0) return APX_OK;
    Scan S = scan_of(a, true);
    APX_SCAN_WORKSPACE();
    APX_REQUIRE(spans_of(S, a, true).apart(), "an output overlaps an input or another output");
    return run(a->type, S, true, a->workspace, (hipStream_t)stream);
}

extern "C" int apx_gated_scan_step(const apx_gated_scan_args* a, float* h, void* stream) {
    APX_REQUIRE(a, "args");
    apx_gated_scan_args one = *a;
    one.T = 1; one.f_t = one.x_t = one.o_t = one.y_t = 0;
    a = &one;
    if (const int rc = check_common(a)) return rc;
    if (a->B == 0 || a->H == 0) return APX_OK;
    APX_REQUIRE(h && aligned(h, 4) && a->B * a->H < ((int64_t)1 << 31), "h, B * H");
    APX_SCAN_IN(f, f); APX_SCAN_IN(x, x); APX_SCAN_OUT(y, y);
    if (a->o) APX_SCAN_IN(o, o);
    const int64_t e = size_of(a->type), row = a->H * e;
    Spans all;
    all.add(span(a->y, 1, 0, a->B, a->y_b * e, row)); all.add(dense(h, a->B * a->H * 4));
    all.outputs = 2;
    // (h itself as f or x is served: what is written is made of what was read there; o is read behind that)
    auto input = [&](const void* p, int64_t sb, bool first) { if (p && !(first && p == h && a->type == APX_F32 && (a->B == 1 || sb == a->H))) all.add(span(p, 1, 0, a->B, sb * e, row)); };
    input(a->f, a->f_b, true); input(a->x, a->x_b, true); input(a->o, a->o_b, false);
    if (a->reset) all.add(dense(a->reset, a->B));
    APX_REQUIRE(all.apart(), "y or h overlaps an input or the other");
    const OneStep S = {a->f, a->x, a->o, a->y, a->f_b * e, a->x_b * e, a->o_b * e, a->y_b * e, a->reset, (unsigned)(a->B * a->H), (unsigned)a->H};
    APX_BY_TYPE(a->type, gated_scan_step_kernel, apx_cdiv(a->B * a->H, 256), 256, (hipStream_t)stream, S, h);
    return APX_OK;
}
