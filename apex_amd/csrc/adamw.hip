// One AdamW step over many tensors behind a global-norm clip, moments in 32 or in 8 bits (include/apx.h, apx_adamw).
//
//   g = k g;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - step m / (sqrt(v) ibc + eps),  step = lr / (1 - b1^t), ibc = 1 / sqrt(1 - b2^t)
//
// Two launches: the first sums the squares of all gradients (one f64 sum per workgroup, its elements in a fixed order) and counts the step, the second adds those sums
// up again in every workgroup - a few kB out of L2, cheaper than a third launch - and makes the step.  Tensors go into the launches by tables in the kernel arguments
// (no device copy of pointers that would have to be kept in step with the caller's): up to TABLE tensors a launch.
// What bounds it: memory for large networks - 28 bytes a parameter with 32-bit moments, 12 + 4 with 8-bit ones, the gradients twice with a clip -, the launches for small ones.
// Measured on an MI355X, 63 M parameters: norm 38 - 70 us (gradients in the caches or not: 3.6 TB/s, what a sum reads at), update 273 us (32 bits, f32 gradients), 168 us (8 bits, bf16
// gradients, 5.3 TB/s); the 450 k parameters of a recurrent actor and critic: 3.8 + 6.2 us.
// Products and sums of the moments are separate roundings (no fused multiply-add), so that the moments are the same numbers wherever the formula above is evaluated in f32.
#include "apx_common.h"
#include <gfx950/half_types.h>
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

namespace {

using namespace half_types;

constexpr int TABLE = 120;                 // entries a launch: 32 bytes each, of 4 kB of kernel arguments
constexpr int BLOCK = 256;                 // elements that share a scale of 8-bit moments, and what a tensor's part of the moments is rounded up to
constexpr int CHUNK = 2048;                // elements a workgroup takes at a time: 8 blocks, 8 elements a thread
constexpr int64_t LARGEST = (int64_t)1 << 39;     // elements of a tensor, and of all
constexpr int64_t ENTRY = (int64_t)1 << 31;      // elements of an entry: a larger tensor takes several
constexpr int PARTS = 1024;                // partial sums of squares of one launch (512 or 2048: 77 and 80 us instead of 73)
constexpr int GRID = 4096;                 // workgroups of the update at most: 16 for each of 256 CUs (8 for each: 335 instead of 323 us, 32 for each: 8-bit moments 5 % slower)
constexpr unsigned M_OFFSET = 904, V_OFFSET = 776;

struct Table {
    float* p[TABLE]; const void* g[TABLE];
    unsigned n[TABLE], state[TABLE];       // elements; the block its moments begin with
    int first[TABLE];                      // its first chunk
    float wd[TABLE];
    int entries, chunks;
};
struct Step { float step, ibc; };

// the entry of a chunk: the last whose first chunk is not beyond it
__device__ __forceinline__ int entry_of(const Table& T, int chunk) {
    int lo = 0, hi = T.entries - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (T.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// 4 elements by one wide access, on any boundary that their type allows (tensors are views at any offset of a flat block)
typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t H4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t C4 __attribute__((aligned(4)));      // 4 codes
template <int TYPE> __device__ __forceinline__ void load_grad(const void* g, int64_t i, float (&o)[4]) {
    if constexpr (TYPE == APX_F32) {
        const F4 r = *(const F4*)((const float*)g + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = r[k];
    } else {
        const H4 r = *(const H4*)((const uint16_t*)g + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = TYPE == APX_BF16 ? widen_bf16(r[k]) : widen_f16(r[k]);
    }
}
template <int TYPE> __device__ __forceinline__ float grad_at(const void* g, int64_t i) {
    if constexpr (TYPE == APX_F32) return ((const float*)g)[i];
    else if constexpr (TYPE == APX_BF16) return widen_bf16(((const uint16_t*)g)[i]);
    else return widen_f16(((const uint16_t*)g)[i]);
}
// up to 4 elements at i of which `have` exist; the others are 0
template <int TYPE> __device__ __forceinline__ void load_grad_end(const void* g, int64_t i, int have, float (&o)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = k < have ? grad_at<TYPE>(g, i + k) : 0.f;
}
// sum over the workgroup's 256 threads in a fixed order; every thread gets it
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return v;
}

__device__ void count_step(int64_t* t, Step* out, double lr, double beta1, double beta2) {
    const int64_t n = *t + 1;
    *t = n;
    out->step = (float)(lr / (1.0 - pow(beta1, (double)n)));
    out->ibc = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)n)));
}
__global__ void adamw_begin_kernel(int64_t* t, Step* out, double lr, double beta1, double beta2) {
    if (threadIdx.x == 0) count_step(t, out, lr, beta1, beta2);
}
template <int TYPE>
__global__ __launch_bounds__(256) void adamw_norm_kernel(Table T, double* parts, int64_t* t, Step* out, double lr, double beta1, double beta2) {
    if (t && blockIdx.x == 0 && threadIdx.x == 0) count_step(t, out, lr, beta1, beta2);
    double sum = 0;
    for (int chunk = blockIdx.x; chunk < T.chunks; chunk += gridDim.x) {
        const int k = entry_of(T, chunk);
        const unsigned e0 = (unsigned)(chunk - T.first[k]) * CHUNK, left = T.n[k] - e0, i = threadIdx.x * 4;
        const void* p = T.g[k];
        float g[2][4];
        if (left >= CHUNK) { load_grad<TYPE>(p, (int64_t)e0 + i, g[0]); load_grad<TYPE>(p, (int64_t)e0 + 1024 + i, g[1]); }
        else { load_grad_end<TYPE>(p, (int64_t)e0 + i, (int)left - (int)i, g[0]); load_grad_end<TYPE>(p, (int64_t)e0 + 1024 + i, (int)left - 1024 - (int)i, g[1]); }
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += (double)g[q >> 2][q & 3] * (double)g[q >> 2][q & 3];
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

struct Hyper {
    float beta1, omb1, beta2, omb2, eps, lr, grad_scale, max_norm; double norm_scale;      // (f64 as the norm is: 1 / 3 in f32 moved it by 3e-8)
    const double* parts; int n_parts;      // 0: no clipping
    const Step* step; const int64_t* t; uint64_t seed; double* norm_out;
};
// What the gradients are multiplied by: k, and 2^-64 before it if `far`; false: the norm is not finite.  Far: the norm, the ratio or k is beyond f32's normal numbers (gradients of 1e37
// in a thousand elements have a norm of 1e39); k is formed in f64 then and taken apart, exactly: a gradient that 2^-64 rounds gives a product below all f32 numbers.
constexpr float LEAST = 1.17549435e-38f;      // the smallest normal number
__device__ __forceinline__ bool clip_factor(const Hyper& P, bool first, float& k, bool& far) {
    k = P.grad_scale; far = false;
    if (P.n_parts == 0) return true;
    double s = 0;
    for (int i = threadIdx.x; i < P.n_parts; i += 256) s += P.parts[i];
    const double norm = sqrt(block_sum(s)) * P.norm_scale;
    if (first && P.norm_out && threadIdx.x == 0) *P.norm_out = norm;
    const float c = P.max_norm / ((float)norm + 1e-6f);
    k = (c < 1.f ? c : 1.f) * P.grad_scale;
    if (c < LEAST || fabsf(k) < LEAST) {
        const double ratio = (double)P.max_norm / (norm + 1e-6), q = (ratio < 1.0 ? ratio : 1.0) * (double)P.grad_scale;
        far = fabs(q) < 0x1p-62;
        k = (float)(far ? q * 0x1p64 : q);
    }
    far = wave_uniform(far);
    return norm <= 1.7976931348623157e308;
}
__device__ __forceinline__ void nearer(float (&g)[2][4]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) g[q >> 2][q & 3] *= 0x1p-64f;
}
__device__ __forceinline__ void adam(float g, float& m, float& v, float& p, const Hyper& P, const Step& S, float keep) {
    m = m * P.beta1 + g * P.omb1;
    v = v * P.beta2 + (g * g) * P.omb2;
    // (fast square root and reciprocal, 1 ulp each: 2e-7 of an update, which is itself a small part of p)
    p = p * keep - S.step * (m * rcp_fast(sqrt_fast(v) * S.ibc + P.eps));
}

// Parameters and moments pass by the caches: nobody reads them again soon, and 63 M parameters' 750 MB would drive out the gradients, which the norm has just brought into the
// 256 MB in front of the memory (ordinary accesses: 320 us for the update of such a network; so: 273 us).
template <int TYPE>
__global__ __launch_bounds__(256) void adamw32_kernel(Table T, Hyper P, float* __restrict__ M, float* __restrict__ V) {
    float c; bool far;      // what a gradient is multiplied by
    if (!clip_factor(P, blockIdx.x == 0, c, far)) return;
    const Step S = *P.step;
    for (int chunk = blockIdx.x; chunk < T.chunks; chunk += gridDim.x) {
        const int id = entry_of(T, chunk);
        const unsigned e0 = (unsigned)(chunk - T.first[id]) * CHUNK, left = T.n[id] - e0;
        float* p = T.p[id] + e0; float* m = M + (int64_t)T.state[id] * BLOCK + e0; float* v = V + (int64_t)T.state[id] * BLOCK + e0;
        const float keep = 1.f - P.lr * T.wd[id];
        if (left >= CHUNK) {
            float g[2][4]; F4 pp[2], mm[2], vv[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = q * 1024 + threadIdx.x * 4;
                load_grad<TYPE>(T.g[id], (int64_t)e0 + i, g[q]);
                pp[q] = APX_PASSING((const F4*)(p + i)); mm[q] = APX_PASSING((const F4*)(m + i)); vv[q] = APX_PASSING((const F4*)(v + i));
            }
            if (far) nearer(g);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int i = q * 1024 + threadIdx.x * 4;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float x = pp[q][k], y = mm[q][k], z = vv[q][k];
                    adam(g[q][k] * c, y, z, x, P, S, keep);
                    pp[q][k] = x; mm[q][k] = y; vv[q][k] = z;
                }
                APX_PASS((F4*)(p + i), pp[q]); APX_PASS((F4*)(m + i), mm[q]); APX_PASS((F4*)(v + i), vv[q]);
            }
        } else {
            for (unsigned i = threadIdx.x; i < left; i += 256) adam(grad_at<TYPE>(T.g[id], (int64_t)e0 + i) * (far ? 0x1p-64f : 1.f) * c, m[i], v[i], p[i], P, S, keep);
        }
    }
}

// ------------------------------------------------------------------------------------------------ 8-bit moments
__device__ __forceinline__ unsigned mix(unsigned x) {      // 32 bits in which every bit of x has a part (a bijection: xor-shifts and odd factors, taken from the square roots of 2 and 3)
    x ^= x >> 16; x *= 0x6A09E667u;
    x ^= x >> 15; x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned step_key(uint64_t seed, int64_t t) {
    return mix(mix((unsigned)seed) ^ mix((unsigned)(seed >> 32) + 0x3C6EF373u) ^ mix((unsigned)t + 0x54FF53A5u));
}
__device__ __forceinline__ unsigned element_noise(unsigned key, int64_t i) { return mix((unsigned)i ^ key ^ ((unsigned)((uint64_t)i >> 32) * 0x3C6EF373u)); }

// s = 2^(the largest's exponent) for a block whose largest |value| has the bits `top`, at least 2^-94 (what the smallest code stands for is a normal number then); NaN for what
// cannot be held
__device__ __forceinline__ void block_scale(unsigned top, float& s, float& inv) {
    unsigned e = top >> 23;
    e = e < 33u ? 33u : e;
    s = __uint_as_float(e << 23); inv = __uint_as_float((254u - e) << 23);
    if (e >= 254) { s = __uint_as_float(0x7fc00000u); inv = 0.f; }
}
constexpr float M_LEAST = 1.125f / (1 << 14), V_LEAST = 1.125f / (1 << 30);      // what c = 1 stands for
__device__ __forceinline__ unsigned encode_m(float m, float inv, unsigned bits16) {
    const float q = fabsf(m) * inv;      // exact: a power of two
    const unsigned r = bits16 << 4;
    unsigned c = ((__float_as_uint(q) + r) >> 20) - M_OFFSET;
    if (q < M_LEAST) c = (float)r * (M_LEAST / (1 << 20)) < q ? 1u : 0u;
    return c | (m < 0.f && c ? 128u : 0u);
}
__device__ __forceinline__ unsigned encode_v(float v, float inv, unsigned bits16) {
    const float q = v * inv;
    unsigned c = ((__float_as_uint(q) + (bits16 << 4)) >> 20) - V_OFFSET;
    if (q < V_LEAST) c = q > 0.f ? 1u : 0u;
    return c;
}
__device__ __forceinline__ float decode_m(unsigned c, float s) {
    const float v = ((c & 127u) ? __uint_as_float(((c & 127u) + M_OFFSET) << 20) : 0.f) * s;
    return (c & 128u) ? -v : v;
}
__device__ __forceinline__ float decode_v(unsigned c, float s) { return (c ? __uint_as_float((c + V_OFFSET) << 20) : 0.f) * s; }

// the largest of a wave's 64 numbers, as a scalar: four exchanges inside the rows of 16 lanes, then the rows' numbers as scalars
__device__ __forceinline__ unsigned wave_top(unsigned x) {
    auto top = [&](int y) { x = x > (unsigned)y ? x : (unsigned)y; };
    top(__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));       // lanes 1 apart
    top(__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));       // 2 apart
    top(__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, true));      // the other half of 8
    top(__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, true));      // the other half of 16
    unsigned r = (unsigned)__builtin_amdgcn_readlane((int)x, 0);
#pragma unroll
    for (int row = 16; row < 64; row += 16) { const unsigned y = (unsigned)__builtin_amdgcn_readlane((int)x, row); r = r > y ? r : y; }
    return r;
}

// A wave takes a block of 256 elements at a time, a lane 4 of them, two blocks of a chunk at once so that twice as many loads are on their way.  Codes and scales are exact in
// f32 (scales are powers of two), the block's largest is found on the bits, so the same inputs give the same codes whatever the launch looks like.
template <int TYPE>
__global__ __launch_bounds__(256) void adamw8_kernel(Table T, Hyper P, uint8_t* __restrict__ M, uint8_t* __restrict__ V, float* __restrict__ MS, float* __restrict__ VS) {
    float c; bool far;      // what a gradient is multiplied by
    if (!clip_factor(P, blockIdx.x == 0, c, far)) return;
    const Step S = *P.step;
    const unsigned key = step_key(P.seed, *P.t);
    const int wave = wave_uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int chunk = blockIdx.x; chunk < T.chunks; chunk += gridDim.x) {
        const int id = entry_of(T, chunk);
        const float keep = 1.f - P.lr * T.wd[id];
        const unsigned n = T.n[id], e0 = (unsigned)(chunk - T.first[id]) * CHUNK;
        float* const p = T.p[id];
        float g[2][4], ms[2], vs[2]; F4 pp[2]; C4 mm[2], vv[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const unsigned e = e0 + (q * 4 + wave) * BLOCK;
            if (e >= n) continue;
            const int64_t blk = (int64_t)T.state[id] + e / BLOCK;
            const unsigned i = e + lane * 4;
            if (n - e >= BLOCK) { load_grad<TYPE>(T.g[id], i, g[q]); pp[q] = APX_PASSING((const F4*)(p + i)); }
            else {
                load_grad_end<TYPE>(T.g[id], i, (int)(n - e) - lane * 4, g[q]);
#pragma unroll
                for (int k = 0; k < 4; ++k) pp[q][k] = i + k < n ? p[i + k] : 0.f;
            }
            mm[q] = APX_PASSING((const C4*)(M + blk * BLOCK + lane * 4)); vv[q] = APX_PASSING((const C4*)(V + blk * BLOCK + lane * 4));
            ms[q] = MS[blk]; vs[q] = VS[blk];
        }
        if (far) nearer(g);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const unsigned e = e0 + (q * 4 + wave) * BLOCK;
            if (e >= n) continue;
            const int64_t blk = (int64_t)T.state[id] + e / BLOCK;
            const unsigned i = e + lane * 4;
            float m[4], v[4];
            unsigned mt = 0, vt = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {      // (behind the tensor's end: codes, gradient and parameter 0 stay 0)
                m[k] = decode_m(mm[q] >> 8 * k & 255u, ms[q]); v[k] = decode_v(vv[q] >> 8 * k & 255u, vs[q]);
                float x = pp[q][k];
                adam(g[q][k] * c, m[k], v[k], x, P, S, keep);
                pp[q][k] = x;
                if (n - e < BLOCK && i + k >= n) m[k] = v[k] = 0.f;      // (0 times an infinite scale factor, say)
                const unsigned am = __float_as_uint(m[k]) & 0x7fffffffu, av = __float_as_uint(v[k]) & 0x7fffffffu;      // (as integers: a NaN is larger than all numbers)
                mt = mt > am ? mt : am; vt = vt > av ? vt : av;
            }
            if (n - e >= BLOCK) APX_PASS((F4*)(p + i), pp[q]);
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k) if (i + k < n) p[i + k] = pp[q][k];
            }
            float s, inv, s2, inv2;
            block_scale(wave_top(mt), s, inv); block_scale(wave_top(vt), s2, inv2);
            C4 mo = 0, vo = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned r = element_noise(key, blk * BLOCK + lane * 4 + k);
                mo |= (encode_m(m[k], inv, r & 0xffffu) & 255u) << 8 * k; vo |= (encode_v(v[k], inv2, r >> 16) & 255u) << 8 * k;
            }
            APX_PASS((C4*)(M + blk * BLOCK + lane * 4), mo); APX_PASS((C4*)(V + blk * BLOCK + lane * 4), vo);
            if (lane == 0) { MS[blk] = s; VS[blk] = s2; }
        }
    }
}

struct alignas(16) Half8 { uint16_t v[8]; };
struct alignas(8) Code8 { uint8_t v[8]; };
// 8 elements a thread: blocks of 256 are whole, and the moments' own buffers are aligned
__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t* __restrict__ M, const uint8_t* __restrict__ V, const float* __restrict__ MS, const float* __restrict__ VS,
                                                            int64_t n, uint16_t* __restrict__ mo, uint16_t* __restrict__ vo) {
    for (int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
        const Code8 m = *(const Code8*)(M + i), v = *(const Code8*)(V + i);
        const float ms = MS[i / BLOCK], vs = VS[i / BLOCK];
        Half8 a, b;
#pragma unroll
        for (int k = 0; k < 8; ++k) { a.v[k] = round_bf16(decode_m(m.v[k], ms)); b.v[k] = round_bf16(decode_v(v.v[k], vs)); }
        *(Half8*)(mo + i) = a; *(Half8*)(vo + i) = b;
    }
}

struct Workspace { Step* step; double* parts; };
Workspace workspace_of(void* w) { return {(Step*)w, (double*)((char*)w + 64)}; }
// `numel` in whole pieces of `by` elements a tensor; sizes that a step refuses count for none
int64_t pieces_of(int n_tensors, const int64_t* numel, int64_t by) {
    int64_t k = 0;
    for (int i = 0; numel && i < n_tensors; ++i) k += numel[i] > 0 && numel[i] < LARGEST ? (numel[i] + by - 1) / by : 0;
    return k;
}
// (one even where there is nothing: it counts the step)
int launches_of(int n_tensors, const int64_t* numel) { const int64_t k = pieces_of(n_tensors, numel, ENTRY); return k ? (int)((k + TABLE - 1) / TABLE) : 1; }

// Does nothing that a step writes - parameters, moments, count, norm, workspace - share memory with anything else that it writes, or with a gradient?  (Gradients may be the same ones.)
// Pieces in the order of their addresses, which sets of tensors mostly have anyway: one walk (a call with 200 tensors takes the host as long as one that only compared base pointers).
struct Piece { uintptr_t from, to; };
bool operator<(const Piece& a, const Piece& b) { return a.from < b.from; }
Piece* in_order(Piece* a, int n) {
    if (!std::is_sorted(a, a + n)) std::sort(a, a + n);
    return a + n;
}
int apart(const apx_adamw_args* a, int64_t elements, size_t workspace) {
    constexpr int FEW = 256;
    Piece few[3 * FEW + 16], rest[8];
    std::unique_ptr<Piece[]> many(a->n_tensors > FEW ? new (std::nothrow) Piece[3 * (size_t)a->n_tensors + 16] : nullptr);
    if (a->n_tensors > FEW && !many) { apx_set_error("apx_adamw: no memory to check %d tensors", a->n_tensors); return APX_E_ARG; }
    Piece* const g = many ? many.get() : few, * const p = g + a->n_tensors, * const w = p + a->n_tensors;
    int ng = 0, np = 0, nr = 0;
    auto piece = [](const void* at, int64_t bytes) { return Piece{(uintptr_t)at, (uintptr_t)at + (uintptr_t)bytes}; };
    for (int i = 0; i < a->n_tensors; ++i) {
        if (a->numel[i] == 0) continue;
        p[np++] = piece(a->params[i], a->numel[i] * 4);
        g[ng++] = piece(a->grads[i], a->numel[i] * (a->grad_type == APX_F32 ? 4 : 2));
    }
    auto add = [&](const void* at, int64_t bytes) { if (at && bytes) rest[nr++] = piece(at, bytes); };
    const int64_t code = a->state_bits == 32 ? 4 : 1;
    add(a->m, elements * code); add(a->v, elements * code);
    if (a->state_bits == 8) { add(a->m_scale, elements / BLOCK * 4); add(a->v_scale, elements / BLOCK * 4); }
    add(a->t, 8); add(a->norm_out, 8); add(a->workspace, (int64_t)workspace);
    in_order(g, ng);
    Piece* const end = std::merge(p, in_order(p, np), rest, in_order(rest, nr), w);
    for (Piece* x = w; x + 1 < end; ++x) APX_REQUIRE(x->to <= x[1].from, "two of the parameters, moments, t, norm_out and workspace overlap");
    const Piece* x = w;
    for (int i = 0; i < ng; ++i) {
        while (x < end && x->to <= g[i].from) ++x;
        APX_REQUIRE(x == end || x->from >= g[i].to, "a gradient lies on what the step writes");
    }
    return APX_OK;
}

}  // namespace

#define APX_BY_TYPE(type, kernel, grid, block, s, ...)                                                                    \
    do {                                                                                                                  \
        if ((type) == APX_F32) hipLaunchKernelGGL(kernel<APX_F32>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);           \
        else if ((type) == APX_BF16) hipLaunchKernelGGL(kernel<APX_BF16>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);    \
        else hipLaunchKernelGGL(kernel<APX_F16>, dim3(grid), dim3(block), 0, s, __VA_ARGS__);                             \
        APX_LAUNCH_CHECK();                                                                                               \
    } while (0)

extern "C" int64_t apx_adamw_state_elements(int n_tensors, const int64_t* numel) {
    return pieces_of(n_tensors, numel, BLOCK) * BLOCK;
}
extern "C" size_t apx_adamw_workspace_bytes(int n_tensors, const int64_t* numel) { return 64 + (size_t)launches_of(n_tensors, numel) * PARTS * sizeof(double); }

extern "C" int apx_adamw(const apx_adamw_args* a, void* stream) {
    APX_REQUIRE(a && a->n_tensors >= 0, "args");
    if (a->n_tensors == 0) return APX_OK;
    APX_REQUIRE(a->params && a->grads && a->numel && a->t, "null pointer");
    APX_REQUIRE((((uintptr_t)a->t | (uintptr_t)a->norm_out) & 7) == 0, "t, norm_out: 8-byte alignment");
    APX_REQUIRE(a->grad_type == APX_F32 || a->grad_type == APX_BF16 || a->grad_type == APX_F16, "grad_type");
    APX_REQUIRE(a->state_bits == 32 || a->state_bits == 8, "state_bits");
    APX_REQUIRE(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1, "beta1, beta2");
    APX_REQUIRE((float)a->eps >= 1.17549435e-38f && std::isfinite((float)a->eps) && std::isfinite((float)a->lr) && std::isfinite((float)a->grad_scale) && !std::isnan(a->max_norm), "eps, lr, grad_scale, max_norm");
    int64_t total = 0;
    for (int i = 0; i < a->n_tensors; ++i) {
        APX_REQUIRE(a->numel[i] >= 0 && a->numel[i] < LARGEST, "numel");
        APX_REQUIRE(a->numel[i] == 0 || (a->params[i] && a->grads[i]), "null tensor");
        APX_REQUIRE(a->numel[i] == 0 || (((uintptr_t)a->params[i] & 3) == 0 && ((uintptr_t)a->grads[i] & (a->grad_type == APX_F32 ? 3 : 1)) == 0), "tensor alignment");
        APX_REQUIRE(!a->weight_decay || std::isfinite(a->weight_decay[i]), "weight_decay");
        total += a->numel[i];
        APX_REQUIRE(total < LARGEST, "numel in all");
    }
    APX_REQUIRE(total == 0 || (a->m && a->v && (a->state_bits == 32 || (a->m_scale && a->v_scale))), "moments");
    APX_REQUIRE((((uintptr_t)a->m | (uintptr_t)a->v | (uintptr_t)a->m_scale | (uintptr_t)a->v_scale) & 3) == 0, "moments: 4-byte alignment");
    const size_t need = apx_adamw_workspace_bytes(a->n_tensors, a->numel);
    APX_REQUIRE(a->workspace && ((uintptr_t)a->workspace & 15) == 0 && a->workspace_bytes >= need, "workspace");
    if (const int rc = apart(a, apx_adamw_state_elements(a->n_tensors, a->numel), need)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    const Workspace W = workspace_of(a->workspace);
    const bool clip = a->max_norm > 0;
    // the entries in order, a launch's worth at a time
    struct Walk { int tensor; int64_t done, state; };
    auto next = [&](Walk& w, Table& T) {
        T.entries = T.chunks = 0;
        while (w.tensor < a->n_tensors && T.entries < TABLE) {
            const int i = w.tensor;
            const int64_t left = a->numel[i] - w.done, n = left < ENTRY ? left : ENTRY;
            if (n > 0) {
                const int k = T.entries++;
                T.p[k] = a->params[i] + w.done;
                T.g[k] = (const char*)a->grads[i] + w.done * (a->grad_type == APX_F32 ? 4 : 2);
                T.n[k] = (unsigned)n; T.state[k] = (unsigned)w.state; T.first[k] = T.chunks;
                T.wd[k] = a->weight_decay ? a->weight_decay[i] : 0.f;
                T.chunks += (int)((n + CHUNK - 1) / CHUNK);
                w.state += (n + BLOCK - 1) / BLOCK;
                w.done += n;
            }
            if (w.done == a->numel[i]) { ++w.tensor; w.done = 0; }
        }
        return T.entries > 0;
    };
    Table T;
    int n_parts = 0;
    if (clip) {
        Walk w = {0, 0, 0};
        for (bool first = true; next(w, T) || first; first = false) {
            const int grid = T.chunks < 1 ? 1 : T.chunks < PARTS ? T.chunks : PARTS;
            APX_BY_TYPE(a->grad_type, adamw_norm_kernel, grid, 256, s, T, W.parts + n_parts, first ? a->t : (int64_t*)nullptr, W.step, a->lr, a->beta1, a->beta2);
            n_parts += grid;
        }
    } else {
        hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(64), 0, s, a->t, W.step, a->lr, a->beta1, a->beta2);
        APX_LAUNCH_CHECK();
    }
    const Hyper P = {(float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2, (float)(1.0 - a->beta2), (float)a->eps, (float)a->lr, (float)a->grad_scale, (float)a->max_norm, std::fabs(a->grad_scale),
                     W.parts, n_parts, W.step, a->t, a->seed, a->norm_out};
    Walk w = {0, 0, 0};
    for (bool first = true; next(w, T) || first; first = false) {      // (a set of empty tensors counts a step and has a norm of 0)
        const int grid = T.chunks < 1 ? 1 : T.chunks < GRID ? T.chunks : GRID;
        Hyper Q = P;
        if (!first) Q.norm_out = nullptr;
        if (a->state_bits == 32) APX_BY_TYPE(a->grad_type, adamw32_kernel, grid, 256, s, T, Q, (float*)a->m, (float*)a->v);
        else APX_BY_TYPE(a->grad_type, adamw8_kernel, grid, 256, s, T, Q, (uint8_t*)a->m, (uint8_t*)a->v, a->m_scale, a->v_scale);
    }
    return APX_OK;
}

extern "C" int apx_adamw_moments(const void* m, const void* v, const float* m_scale, const float* v_scale, int64_t elements, void* m_out, void* v_out, void* stream) {
    APX_REQUIRE(elements >= 0 && elements % BLOCK == 0, "elements: whole blocks of 256");
    if (elements == 0) return APX_OK;
    APX_REQUIRE(m && v && m_scale && v_scale && m_out && v_out, "null pointer");
    APX_REQUIRE((((uintptr_t)m_scale | (uintptr_t)v_scale) & 3) == 0 && (((uintptr_t)m | (uintptr_t)v) & 7) == 0 && (((uintptr_t)m_out | (uintptr_t)v_out) & 15) == 0, "alignment");
    const Piece io[6] = {{(uintptr_t)m_out, (uintptr_t)m_out + 2 * (uintptr_t)elements}, {(uintptr_t)v_out, (uintptr_t)v_out + 2 * (uintptr_t)elements},
                         {(uintptr_t)m, (uintptr_t)m + (uintptr_t)elements}, {(uintptr_t)v, (uintptr_t)v + (uintptr_t)elements},
                         {(uintptr_t)m_scale, (uintptr_t)m_scale + (uintptr_t)(elements / BLOCK * 4)}, {(uintptr_t)v_scale, (uintptr_t)v_scale + (uintptr_t)(elements / BLOCK * 4)}};
    for (int i = 0; i < 2; ++i) for (int k = i + 1; k < 6; ++k) APX_REQUIRE(io[i].to <= io[k].from || io[k].to <= io[i].from, "an output overlaps an input or the other output");
    const int64_t want = (elements + 2047) / 2048;
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)(want < GRID ? want : GRID)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)m, (const uint8_t*)v, m_scale, v_scale,
                       elements, (uint16_t*)m_out, (uint16_t*)v_out);
    APX_LAUNCH_CHECK();
    return APX_OK;
}
