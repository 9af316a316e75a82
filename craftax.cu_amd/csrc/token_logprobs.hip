// Log-probabilities of given tokens (actions) with the entropy of each row's distribution and
// its most probable alternatives, and the gradient of all three with respect to the logits.
// No counterpart in the reference, whose head kernels (k_value_sample, craftax_full.cu:9714;
// k_head_bwd_win, :9603) are fixed to the 43 actions it samples itself.
//
// Row of logits x_v, v in the allowed set (mask byte not 0 and x_v > -inf), given token t:
//   m = max x_v,  s = sum e^(x_v - m),  lp = (x_t - m) - ln s,  p_v = e^(x_v - m) / s,
//   H = ln s - (1/s) sum e^(x_v - m) (x_v - m)
// and with incoming gradients g (of lp), h (of H), a_j (of the j-th alternative's lp):
//   dx_v = g [v = t] + sum_j a_j [v = id_j] - p_v (g + sum_j a_j + h (ln p_v + H)).
// The forward reads the logits once (running maximum and sums, rescaled when the maximum
// grows), the gradient reads them once and writes as many values: both are bound by HBM.
// lp is taken from x_t - m and ln s, never from x_t - (m + ln s): with logits of 1e4 the sum
// m + ln s has lost the bits of ln s.  All sums are fp32 per lane (at most a few hundred terms
// each, in [0, 1]) and joined in a tree of fixed shape: the same call gives the same bits.
#include <float.h>

#include "cfp_internal.h"

namespace cfp {
namespace {

constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// Exponents below this give e = 0 in fp32 with hundreds of binades to spare; products e * y are
// taken with y clamped here so that e = 0 never meets y = -inf.
constexpr float kFar = -1.0e4f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }

// 16 bytes of a row that is aligned to its element only (rows of odd width): one
// global_load_dwordx4, which gfx950 issues at any byte address.
template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
    Vec<T> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) {
    __builtin_memcpy(p, &r, sizeof r);
}

// ---- running softmax sums of one lane ------------------------------------------------
// m starts at the lowest finite number instead of -inf: x - m is then never -inf - -inf, and a
// row of the type's lowest values still counts its entries (e^0).  s = 0 at the end: nothing
// was allowed.  u = sum e * y with y = (x - m) log2 e.
struct Sums {
    float m = -FLT_MAX, s = 0.0f, u = 0.0f;
};
__device__ __forceinline__ void raise_max(Sums& a, float m) {
    const float y = fmaxf((a.m - m) * kLog2e, kFar);
    const float r = __builtin_amdgcn_exp2f(y);
    a.u = r * (a.u + a.s * y);
    a.s *= r;
    a.m = m;
}
__device__ __forceinline__ void add_entry(Sums& a, float x) {
    const float y = (x - a.m) * kLog2e;
    const float e = __builtin_amdgcn_exp2f(y);   // NaN stays NaN; results below 2^-126 are 0
    a.s += e;
    a.u += e * fmaxf(y, kFar);
}
__device__ __forceinline__ void join(Sums& a, float m, float s, float u) {
    const float top = fmaxf(a.m, m);
    raise_max(a, top);
    Sums b;
    b.m = m; b.s = s; b.u = u;
    raise_max(b, top);
    a.s += b.s;
    a.u += b.u;
}
// all-reduce over `width` consecutive lanes (a power of two)
template <int WIDTH>
__device__ __forceinline__ void join_lanes(Sums& a) {
    float top = a.m;
#pragma unroll
    for (int d = WIDTH / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, WIDTH));
    raise_max(a, top);
#pragma unroll
    for (int d = WIDTH / 2; d > 0; d >>= 1) {
        a.s += __shfl_xor(a.s, d, WIDTH);
        a.u += __shfl_xor(a.u, d, WIDTH);
    }
}

// ---- the best `top` entries seen by one wavefront -----------------------------------
// Lane i holds the entry of rank i (value, index), best first; -1 marks a free place.  Order:
// larger value, then lower index.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
struct Best {
    float v = -INFINITY;
    int i = -1;
    float last_v = -INFINITY;   // the entry of rank top - 1: what a newcomer has to beat
    int last_i = -1;
    // wave-uniform (nv, ni)
    __device__ __forceinline__ void insert(float nv, int ni, int top) {
        const int lane = (int)(threadIdx.x & 63);
        const int pos = __popcll(__ballot(before(v, i, nv, ni)));
        const float pv = __shfl_up(v, 1);
        const int pi = __shfl_up(i, 1);
        if (lane > pos) { v = pv; i = pi; }
        if (lane == pos) { v = nv; i = ni; }
        last_v = lane_value(v, top - 1);
        last_i = __builtin_amdgcn_readlane(i, top - 1);
    }
    // one entry a lane (wave-uniform call); entries of -inf and NaN never enter: the free
    // places compare as (-inf, -1), which nothing of value -inf comes before
    __device__ __forceinline__ void offer(float x, int idx, int top) {
        unsigned long long todo = __ballot(before(x, idx, last_v, last_i));
        while (todo) {
            const int l = __ffsll(todo) - 1;
            todo &= todo - 1;
            const float nv = lane_value(x, l);
            const int ni = __builtin_amdgcn_readlane(idx, l);
            if (before(nv, ni, last_v, last_i)) insert(nv, ni, top);
        }
    }
};

struct LpArgs {
    const void* x;
    int64_t ld;
    int rows, vocab;
    const int32_t* tok;
    const uint8_t* mask;   // or null
    int64_t ld_mask;       // 0: one mask for all rows
    float* lp;
    float* ent;            // or null
    int top;
    int32_t* ids;
    float* top_lp;
    float* stats;          // [rows][3] or null
    int splits, chunk;     // entries per split, a multiple of 8
    f4* part;              // [rows][splits] (m, s, u, -)
    float2* part_top;      // [rows][splits][top] (value, index bits)
};

// Outputs of one row from its sums; called by one lane.  xt: the given token's logit, -inf
// where it is not allowed.
__device__ __forceinline__ void write_row(const LpArgs& a, int row, const Sums& z, int tok, float xt) {
    const bool none = z.s == 0.0f;
    const float ls = none ? INFINITY : logf(z.s);
    float lp = none ? -INFINITY : (xt - z.m) - ls;
    if (tok < 0) lp = 0.0f;
    else if (tok >= a.vocab || z.s != z.s) lp = NAN;
    a.lp[row] = lp;
    const float h = none ? 0.0f : ls - z.u / z.s * kLn2;
    if (a.ent) a.ent[row] = h;
    if (a.stats) {
        float* st = a.stats + (size_t)row * 3;
        st[0] = none ? 0.0f : z.m;
        st[1] = ls;
        st[2] = h;
    }
}
__device__ __forceinline__ void write_top(const LpArgs& a, int row, const Sums& z, int rank, float v, int i) {
    const size_t o = (size_t)row * a.top + rank;
    const bool bad = z.s != z.s;   // NaN or +inf among the allowed entries
    a.ids[o] = bad ? -1 : i;
    a.top_lp[o] = bad ? NAN : i < 0 ? -INFINITY : (v - z.m) - logf(z.s);
}
template <typename T>
__device__ __forceinline__ float token_logit(const LpArgs& a, int row, int tok) {
    if (tok < 0 || tok >= a.vocab) return -INFINITY;
    const float x = to_f32(((const T*)a.x)[(size_t)row * a.ld + tok]);
    if (a.mask && a.mask[(size_t)row * a.ld_mask + tok] == 0) return -INFINITY;
    return x;
}

// ---- short rows: L lanes a row, up to four entries a lane -----------------------------
// Each load instruction of a lane group covers L consecutive entries of its row.  No online
// rescaling: the row sits in registers.  kShortMax entries at most.
constexpr int kShortR = 4;
constexpr int kShortMax = 64 * kShortR;
template <typename T, int L, bool MASK>
__global__ __launch_bounds__(256) void k_logprobs_short(LpArgs a) {
    const int sub = threadIdx.x % L;
    const int per = 256 / L;
    for (int row0 = (int)blockIdx.x * per; row0 < a.rows; row0 += (int)gridDim.x * per) {
        const int row = row0 + (int)threadIdx.x / L;
        const bool live = row < a.rows;
        const int r = live ? row : a.rows - 1;
        const T* x = (const T*)a.x + (size_t)r * a.ld;
        const uint8_t* mask = MASK ? a.mask + (size_t)r * a.ld_mask : nullptr;
        const int tok = a.tok[r];
        const float xt = token_logit<T>(a, r, tok);
        float v[kShortR];
        Sums z;
#pragma unroll
        for (int j = 0; j < kShortR; j++) {
            const int i = j * L + sub;
            v[j] = -INFINITY;
            if (i < a.vocab && (!MASK || mask[i])) v[j] = to_f32(x[i]);
            z.m = fmaxf(z.m, v[j]);
        }
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) z.m = fmaxf(z.m, __shfl_xor(z.m, d, L));
#pragma unroll
        for (int j = 0; j < kShortR; j++) add_entry(z, v[j]);
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) {
            z.s += __shfl_xor(z.s, d, L);
            z.u += __shfl_xor(z.u, d, L);
        }
        if (live && sub == 0) write_row(a, row, z, tok, xt);
        for (int k = 0; k < a.top; k++) {   // wave-uniform trip count
            float bv = -INFINITY;
            int bi = -1;
#pragma unroll
            for (int j = 0; j < kShortR; j++)   // ascending index: ties keep the first
                if (v[j] > bv) { bv = v[j]; bi = j * L + sub; }
#pragma unroll
            for (int d = L / 2; d > 0; d >>= 1) {
                const float ov = __shfl_xor(bv, d, L);
                const int oi = __shfl_xor(bi, d, L);
                if (before(ov, oi, bv, bi)) { bv = ov; bi = oi; }
            }
#pragma unroll
            for (int j = 0; j < kShortR; j++)
                if (j * L + sub == bi) v[j] = -INFINITY;
            if (live && sub == 0) write_top(a, row, z, k, bv, bi);
        }
    }
}

// ---- long rows -------------------------------------------------------------------------
// One tile: U vectors a lane, all loads in flight before the first use.
constexpr int kU = 4;
template <typename T, bool MASK, bool TOP>
__device__ __forceinline__ void take_tile(const float (&v)[kU][Vec<T>::N], int i0, int vec_stride, Sums& z,
                                          Best& best, int top) {
    constexpr int N = Vec<T>::N;
    float tm = v[0][0];
#pragma unroll
    for (int q = 0; q < kU; q++)
#pragma unroll
        for (int j = 0; j < N; j++) tm = fmaxf(tm, v[q][j]);
    if (tm > z.m) raise_max(z, tm);
#pragma unroll
    for (int q = 0; q < kU; q++)
#pragma unroll
        for (int j = 0; j < N; j++) add_entry(z, v[q][j]);
    if (TOP && __any(tm >= best.last_v && tm > -INFINITY)) {
#pragma unroll
        for (int q = 0; q < kU; q++)
#pragma unroll
            for (int j = 0; j < N; j++) best.offer(v[q][j], i0 + q * vec_stride + j, top);
    }
}

// W wavefronts of a workgroup stream entries [lo, hi) of a row; thread t takes vectors t,
// t + 64 W, ...  Every wavefront runs the same number of tiles (uniform trip count).
template <typename T, bool MASK, bool TOP, int W>
__device__ __forceinline__ void stream_row(const T* x, const uint8_t* mask, int lo, int hi, Sums& z, Best& best,
                                           int top) {
    constexpr int N = Vec<T>::N, STRIDE = 64 * W * N, TILE = STRIDE * kU;
    const int t = W == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    int base = lo;
    float v[kU][N];
    for (; base + TILE <= hi; base += TILE) {
        const int i0 = base + t * N;
        Vec<T> raw[kU];
        uint8_t mk[kU][N];
#pragma unroll
        for (int q = 0; q < kU; q++) {
            raw[q] = load_vec(x + i0 + q * STRIDE);
            if (MASK) __builtin_memcpy(mk[q], mask + i0 + q * STRIDE, N);
        }
#pragma unroll
        for (int q = 0; q < kU; q++)
#pragma unroll
            for (int j = 0; j < N; j++) {
                v[q][j] = to_f32(raw[q].v[j]);
                if (MASK && mk[q][j] == 0) v[q][j] = -INFINITY;
            }
        take_tile<T, MASK, TOP>(v, i0, STRIDE, z, best, top);
    }
    if (base < hi) {   // the last, partial tile: whole vectors where they fit, entries at the end
        const int i0 = base + t * N;
#pragma unroll
        for (int q = 0; q < kU; q++) {
            const int i = i0 + q * STRIDE;
            if (i + N <= hi) {
                const Vec<T> raw = load_vec(x + i);
                uint8_t mk[N];
                if (MASK) __builtin_memcpy(mk, mask + i, N);
#pragma unroll
                for (int j = 0; j < N; j++) v[q][j] = MASK && mk[j] == 0 ? -INFINITY : to_f32(raw.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    v[q][j] = -INFINITY;
                    if (i + j < hi && (!MASK || mask[i + j])) v[q][j] = to_f32(x[i + j]);
                }
            }
        }
        take_tile<T, MASK, TOP>(v, i0, STRIDE, z, best, top);
    }
}

// One wavefront a row, four rows a workgroup: rows that are many or not long.
template <typename T, bool MASK, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_wave(LpArgs a) {
    const int lane = threadIdx.x & 63;
    for (int row0 = (int)blockIdx.x * 4; row0 < a.rows; row0 += (int)gridDim.x * 4) {
        const int row = row0 + (int)(threadIdx.x >> 6);
        if (row >= a.rows) return;   // whole wavefronts; nothing below synchronises a workgroup
        const int tok = a.tok[row];
        const float xt = token_logit<T>(a, row, tok);
        Sums z;
        Best best;
        stream_row<T, MASK, TOP, 1>((const T*)a.x + (size_t)row * a.ld,
                                    MASK ? a.mask + (size_t)row * a.ld_mask : nullptr, 0, a.vocab, z, best, a.top);
        join_lanes<64>(z);
        if (lane == 0) write_row(a, row, z, tok, xt);
        if (TOP && lane < a.top) write_top(a, row, z, lane, best.v, best.i);
    }
}

// One workgroup for entries [split * chunk, ...) of a row; with one split it writes the
// outputs, else its part, which k_logprobs_join puts together.
constexpr int kWaves = 4;
template <typename T, bool MASK, bool TOP>
__global__ __launch_bounds__(64 * kWaves) void k_logprobs_group(LpArgs a) {
    __shared__ float zs[kWaves][3];
    __shared__ float2 lists[kWaves][kMaxTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
    const int lo = split * a.chunk, hi = lo + a.chunk < a.vocab ? lo + a.chunk : a.vocab;
    const int tok = a.tok[row];
    const float xt = a.splits == 1 ? token_logit<T>(a, row, tok) : 0.0f;
    Sums z;
    Best best;
    stream_row<T, MASK, TOP, kWaves>((const T*)a.x + (size_t)row * a.ld,
                                     MASK ? a.mask + (size_t)row * a.ld_mask : nullptr, lo, hi, z, best, a.top);
    join_lanes<64>(z);
    if (lane == 0) { zs[wave][0] = z.m; zs[wave][1] = z.s; zs[wave][2] = z.u; }
    if (TOP && wave > 0 && lane < a.top) lists[wave][lane] = make_float2(best.v, __int_as_float(best.i));
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; w++) join(z, zs[w][0], zs[w][1], zs[w][2]);
    if (TOP)
        for (int w = 1; w < kWaves; w++) {
            const float2 e = lane < a.top ? lists[w][lane] : make_float2(-INFINITY, __int_as_float(-1));
            best.offer(e.x, __float_as_int(e.y), a.top);
        }
    if (a.splits == 1) {
        if (lane == 0) write_row(a, row, z, tok, xt);
        if (TOP && lane < a.top) write_top(a, row, z, lane, best.v, best.i);
        return;
    }
    const size_t o = (size_t)row * a.splits + split;
    if (lane == 0) a.part[o] = f4{z.m, z.s, z.u, 0.0f};
    if (TOP && lane < a.top) a.part_top[o * a.top + lane] = make_float2(best.v, __int_as_float(best.i));
}

// One wavefront a row: the parts of its splits in ascending order of lane, then the tree.
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_join(LpArgs a) {
    const int lane = threadIdx.x, row = (int)blockIdx.x;
    const int tok = a.tok[row];
    const float xt = token_logit<T>(a, row, tok);
    Sums z;
    for (int s = lane; s < a.splits; s += 64) {
        const f4 p = a.part[(size_t)row * a.splits + s];
        join(z, p[0], p[1], p[2]);
    }
    join_lanes<64>(z);
    if (lane == 0) write_row(a, row, z, tok, xt);
    if (a.top > 0) {
        Best best;
        const int total = a.splits * a.top;
        for (int o = 0; o < total; o += 64) {
            float2 e = make_float2(-INFINITY, __int_as_float(-1));
            if (o + lane < total) e = a.part_top[(size_t)row * total + o + lane];
            best.offer(e.x, __float_as_int(e.y), a.top);
        }
        if (lane < a.top) write_top(a, row, z, lane, best.v, best.i);
    }
}

// ---- gradient ---------------------------------------------------------------------------
struct LpGradArgs {
    const void* x;         // not restrict: dx may be x itself
    int64_t ld;
    int rows, vocab;
    const int32_t* tok;
    const uint8_t* mask;
    int64_t ld_mask;
    const float* stats;
    const float* g_lp;     // or null
    const float* g_ent;    // or null
    int top;               // 0: no gradient from the alternatives
    const int32_t* ids;
    const float* g_top;
    void* dx;
    int64_t ld_dx;
    int splits, chunk;
};
// What a row's entries share.
struct RowGrad {
    float m, ls, h, weight, g_ent;
    bool none;   // nothing allowed: the gradient is zero whatever comes in
    __device__ __forceinline__ float at(float x) const {
        const float l = (x - m) - ls;
        const float p = __builtin_amdgcn_exp2f(l * kLog2e);
        return -p * (weight + g_ent * (fmaxf(l, kFar) + h));
    }
};
template <typename T>
__device__ __forceinline__ bool entry_allowed(const LpGradArgs& a, int row, int i) {
    return (!a.mask || a.mask[(size_t)row * a.ld_mask + i]) &&
           !(to_f32(((const T*)a.x)[(size_t)row * a.ld + i]) == -INFINITY);
}
// The j-th named entry of a row: j = 0 the given token, 1 .. top the alternatives.  Its index
// (-1: takes no part) and its incoming gradient; an index past the row poisons the row.
template <typename T>
__device__ __forceinline__ int named_entry(const LpGradArgs& a, int row, int j, float& g) {
    g = 0.0f;
    if (j == 0 ? !a.g_lp : j > a.top) return -1;
    const int i = j == 0 ? a.tok[row] : a.ids[(size_t)row * a.top + j - 1];
    if (i < 0) return -1;
    if (i >= a.vocab) { g = NAN; return -1; }
    if (!entry_allowed<T>(a, row, i)) return -1;
    g = j == 0 ? a.g_lp[row] : a.g_top[(size_t)row * a.top + j - 1];
    return i;
}
__device__ __forceinline__ void row_grad(const LpGradArgs& a, int row, float weight, RowGrad& r) {
    const float* st = a.stats + (size_t)row * 3;
    r.m = st[0]; r.ls = st[1]; r.h = st[2];
    r.none = r.ls == INFINITY;
    r.weight = weight;
    r.g_ent = a.g_ent ? a.g_ent[row] : 0.0f;
}
template <int WIDTH>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
    for (int d = WIDTH / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, WIDTH);
    return v;
}

template <typename T, int L, bool MASK>
__global__ __launch_bounds__(256) void k_logprobs_grad_short(LpGradArgs a) {
    const int sub = threadIdx.x % L;
    const int per = 256 / L;
    for (int row0 = (int)blockIdx.x * per; row0 < a.rows; row0 += (int)gridDim.x * per) {
        const int row = row0 + (int)threadIdx.x / L;
        const bool live = row < a.rows;
        const int r = live ? row : a.rows - 1;
        const T* x = (const T*)a.x + (size_t)r * a.ld;
        const uint8_t* mask = MASK ? a.mask + (size_t)r * a.ld_mask : nullptr;
        float v[kShortR], d[kShortR];
        float weight = 0.0f;
#pragma unroll
        for (int j = 0; j < kShortR; j++) {
            const int i = j * L + sub;
            v[j] = -INFINITY;
            if (i < a.vocab && (!MASK || mask[i])) v[j] = to_f32(x[i]);
            d[j] = 0.0f;
        }
        for (int j = 0; j <= a.top; j++) {
            float g;
            const int i = named_entry<T>(a, r, j, g);
            weight += g;
#pragma unroll
            for (int q = 0; q < kShortR; q++)
                if (q * L + sub == i) d[q] += g;
        }
        RowGrad rg;
        row_grad(a, r, weight, rg);
        T* dx = (T*)a.dx + (size_t)r * a.ld_dx;
#pragma unroll
        for (int j = 0; j < kShortR; j++) {
            const int i = j * L + sub;
            const bool on = !rg.none && !(v[j] == -INFINITY);
            // every load of this row was used above: the row may be overwritten in place
            if (live && i < a.vocab) dx[i] = (T)(on ? rg.at(v[j]) + d[j] : 0.0f);
        }
    }
}

// Entries [lo, hi) of a row by one workgroup: what all entries have in common first, then the
// named entries (given token, alternatives) once more by one lane each.  Their logits are read
// before the first store, their values stored behind the last one (barriers on both sides), so
// that dx may be x.
template <typename T, bool MASK>
__global__ __launch_bounds__(256) void k_logprobs_grad(LpGradArgs a) {
    constexpr int N = Vec<T>::N, STRIDE = 256 * N, TILE = STRIDE * kU;
    const int row = (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
    const int lo = split * a.chunk, hi = lo + a.chunk < a.vocab ? lo + a.chunk : a.vocab;
    const T* x = (const T*)a.x + (size_t)row * a.ld;
    const uint8_t* mask = MASK ? a.mask + (size_t)row * a.ld_mask : nullptr;
    T* dx = (T*)a.dx + (size_t)row * a.ld_dx;
    const int lane = threadIdx.x & 63;
    // every wavefront holds all named entries, one a lane (top <= 32)
    float g;
    const int named = named_entry<T>(a, row, lane, g);
    RowGrad rg;
    row_grad(a, row, sum_lanes<64>(g), rg);
    float patch = 0.0f;
    const bool mine = threadIdx.x < 64 && named >= lo && named < hi && !rg.none;
    if (threadIdx.x < 64) {
        patch = mine ? rg.at(to_f32(x[named])) : 0.0f;
        for (int j = 0; j <= a.top; j++)   // an index that is named twice gets both gradients
            if (__builtin_amdgcn_readlane(named, j) == named)
                patch += lane_value(g, j);
    }
    __syncthreads();
    int base = lo;
    for (; base + TILE <= hi; base += TILE) {
        const int i0 = base + (int)threadIdx.x * N;
        Vec<T> raw[kU];
        uint8_t mk[kU][N];
#pragma unroll
        for (int q = 0; q < kU; q++) {
            raw[q] = load_vec(x + i0 + q * STRIDE);
            if (MASK) __builtin_memcpy(mk[q], mask + i0 + q * STRIDE, N);
        }
#pragma unroll
        for (int q = 0; q < kU; q++) {
            Vec<T> out;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float xv = to_f32(raw[q].v[j]);
                const bool on = !rg.none && !(MASK && mk[q][j] == 0) && !(xv == -INFINITY);
                out.v[j] = (T)(on ? rg.at(xv) : 0.0f);
            }
            store_vec(dx + i0 + q * STRIDE, out);
        }
    }
    for (int i = base + (int)threadIdx.x; i < hi; i += 256) {
        const float xv = to_f32(x[i]);
        const bool on = !rg.none && !(MASK && mask[i] == 0) && !(xv == -INFINITY);
        dx[i] = (T)(on ? rg.at(xv) : 0.0f);
    }
    __syncthreads();
    if (mine) dx[named] = (T)patch;
}

// ---- plans --------------------------------------------------------------------------------
struct LpPlan {
    int kind;     // 0 short, 1 a wavefront a row, 2 a workgroup a split
    int splits, chunk;
};
// Rows of up to 256 entries sit in the registers of 16 or 64 lanes.  Longer ones are streamed: by
// a wavefront each where there are enough rows to fill the machine that way (256 CUs, 16
// wavefronts each) and a row is not so long that its last wavefronts run alone; by a workgroup
// each otherwise, split further until about four workgroups a CU run, none with less than 4096
// entries (one tile of 16-bit loads is 8192, and a second launch joins the parts).
LpPlan plan_forward(int rows, int vocab) {
    if (vocab <= kShortMax) return {0, 1, 0};
    if (rows >= 4096 && vocab <= 8192) return {1, 1, 0};
    const int want = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    const int most = (vocab + 4095) / 4096;
    int splits = want < most ? want : most;
    const int chunk = ((vocab + splits - 1) / splits + 7) / 8 * 8;
    splits = (vocab + chunk - 1) / chunk;
    return {2, splits, chunk};
}
// the gradient's parts are independent: 16384 entries a workgroup at most, 2048 at least
LpPlan plan_grad(int rows, int vocab) {
    if (vocab <= kShortMax) return {0, 1, 0};
    int splits = (vocab + 16383) / 16384;
    while ((int64_t)rows * splits < 2048 && (vocab + splits - 1) / splits > 2048) splits *= 2;
    const int chunk = ((vocab + splits - 1) / splits + 7) / 8 * 8;
    return {2, (vocab + chunk - 1) / chunk, chunk};
}
size_t part_bytes(int rows, int splits, int top) {
    return splits == 1 ? 0 : (size_t)rows * splits * (sizeof(f4) + (size_t)top * sizeof(float2));
}

constexpr int kMaxVocab = 1 << 30;
// workgroups of a launch: threads of a grid are counted in 32 bits
constexpr int64_t kMaxGroups = ((int64_t)1 << 32) / 256 - 1;
int capped_groups(int64_t g) { return (int)(g < kMaxGroups ? g : kMaxGroups); }

template <typename T, bool MASK>
void run_forward(const LpArgs& a, const LpPlan& pl, hipStream_t st) {
    if (pl.kind == 0) {
        if (a.vocab <= 16 * kShortR)
            hipLaunchKernelGGL((k_logprobs_short<T, 16, MASK>), dim3(capped_groups(((int64_t)a.rows + 15) / 16)),
                               dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((k_logprobs_short<T, 64, MASK>), dim3(capped_groups(((int64_t)a.rows + 3) / 4)),
                               dim3(256), 0, st, a);
    } else if (pl.kind == 1) {
        const dim3 grid(capped_groups(((int64_t)a.rows + 3) / 4));
        if (a.top > 0) hipLaunchKernelGGL((k_logprobs_wave<T, MASK, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_logprobs_wave<T, MASK, false>), grid, dim3(256), 0, st, a);
    } else {
        const dim3 grid((unsigned)((int64_t)a.rows * a.splits));
        if (a.top > 0) hipLaunchKernelGGL((k_logprobs_group<T, MASK, true>), grid, dim3(64 * kWaves), 0, st, a);
        else hipLaunchKernelGGL((k_logprobs_group<T, MASK, false>), grid, dim3(64 * kWaves), 0, st, a);
        if (a.splits > 1) hipLaunchKernelGGL(k_logprobs_join<T>, dim3(a.rows), dim3(64), 0, st, a);
    }
}
template <typename T, bool MASK>
void run_grad(const LpGradArgs& a, const LpPlan& pl, hipStream_t st) {
    if (pl.kind == 0) {
        if (a.vocab <= 16 * kShortR)
            hipLaunchKernelGGL((k_logprobs_grad_short<T, 16, MASK>),
                               dim3(capped_groups(((int64_t)a.rows + 15) / 16)), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((k_logprobs_grad_short<T, 64, MASK>),
                               dim3(capped_groups(((int64_t)a.rows + 3) / 4)), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((k_logprobs_grad<T, MASK>), dim3((unsigned)((int64_t)a.rows * a.splits)), dim3(256), 0,
                           st, a);
    }
}

int check_rows(const char* who, int dtype, const void* x, int64_t ld, int rows, int vocab, const int32_t* tok,
               const uint8_t* mask, int64_t ld_mask, int top) {
    CFP_REQUIRE(dtype == CFP_F32 || dtype == CFP_BF16 || dtype == CFP_F16, "%s: dtype must be CFP_F32, CFP_BF16 or CFP_F16 (got %d)",
                who, dtype);
    CFP_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= kMaxVocab, "%s: rows must not be negative and vocab in 1..2^30 (got %d, %d)",
                who, rows, vocab);
    CFP_REQUIRE(top >= 0 && top <= kMaxTop, "%s: top must be in 0..%d (got %d)", who, kMaxTop, top);
    if (rows == 0) return 0;
    CFP_REQUIRE(x && tok, "%s: NULL logits or tokens", who);
    CFP_REQUIRE(ld >= vocab || (rows == 1 && ld >= 0), "%s: rows of %d logits need a stride of at least that (got %lld)", who, vocab,
                (long long)ld);
    CFP_REQUIRE(!mask || ld_mask == 0 || ld_mask >= vocab || rows == 1,
                "%s: the mask's row stride must be 0 (one mask for all rows) or at least vocab (got %lld)", who,
                (long long)ld_mask);
    CFP_REQUIRE((reinterpret_cast<uintptr_t>(x) & (dtype == CFP_F32 ? 3u : 1u)) == 0, "%s: logits not aligned to their type", who);
    return 0;
}
size_t elem_bytes(int dtype) { return dtype == CFP_F32 ? 4 : 2; }

}  // namespace
}  // namespace cfp

using namespace cfp;

extern "C" {

size_t cfp_token_logprobs_workspace(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab || top < 0 || top > kMaxTop) return 0;
    return part_bytes(rows, plan_forward(rows, vocab).splits, top);
}

int cfp_token_logprobs(const void* d_logits, int dtype, int64_t ld, int rows, int vocab, const int32_t* d_tokens,
                       const uint8_t* d_mask, int64_t ld_mask, float* d_logprobs, float* d_entropy, int top,
                       int32_t* d_top_ids, float* d_top_logprobs, float* d_stats, void* d_work,
                       size_t work_bytes, void* stream) {
    if (check_rows("cfp_token_logprobs", dtype, d_logits, ld, rows, vocab, d_tokens, d_mask, ld_mask, top)) return 1;
    if (rows == 0) return 0;
    CFP_REQUIRE(d_logprobs, "cfp_token_logprobs: NULL output");
    CFP_REQUIRE(top == 0 || (d_top_ids && d_top_logprobs), "cfp_token_logprobs: top = %d needs both arrays of alternatives", top);
    const LpPlan pl = plan_forward(rows, vocab);
    CFP_REQUIRE(pl.kind < 2 || (int64_t)rows * pl.splits <= kMaxGroups, "cfp_token_logprobs: %d rows of %d are more than one launch holds",
                rows, vocab);
    const size_t need = part_bytes(rows, pl.splits, top);
    CFP_REQUIRE(need == 0 || (d_work && work_bytes >= need && (reinterpret_cast<uintptr_t>(d_work) & 15u) == 0),
                "cfp_token_logprobs: needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, work_bytes);
    LpArgs a{};
    a.x = d_logits; a.ld = ld; a.rows = rows; a.vocab = vocab; a.tok = d_tokens;
    a.mask = d_mask; a.ld_mask = ld_mask;
    a.lp = d_logprobs; a.ent = d_entropy; a.top = top; a.ids = d_top_ids; a.top_lp = d_top_logprobs;
    a.stats = d_stats;
    a.splits = pl.splits; a.chunk = pl.chunk;
    a.part = (f4*)d_work;
    a.part_top = need ? (float2*)((f4*)d_work + (size_t)rows * pl.splits) : nullptr;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == CFP_F32) { d_mask ? run_forward<float, true>(a, pl, st) : run_forward<float, false>(a, pl, st); }
    else if (dtype == CFP_BF16) { d_mask ? run_forward<__bf16, true>(a, pl, st) : run_forward<__bf16, false>(a, pl, st); }
    else { d_mask ? run_forward<_Float16, true>(a, pl, st) : run_forward<_Float16, false>(a, pl, st); }
    CFP_HIP_TRY(hipGetLastError());
    return 0;
}

int cfp_token_logprobs_grad(const void* d_logits, int dtype, int64_t ld, int rows, int vocab,
                            const int32_t* d_tokens, const uint8_t* d_mask, int64_t ld_mask,
                            const float* d_stats, const float* d_g_logprobs, const float* d_g_entropy, int top,
                            const int32_t* d_top_ids, const float* d_g_top, void* d_dlogits, int64_t ld_dlogits,
                            void* stream) {
    if (check_rows("cfp_token_logprobs_grad", dtype, d_logits, ld, rows, vocab, d_tokens, d_mask, ld_mask, top)) return 1;
    if (rows == 0) return 0;
    CFP_REQUIRE(d_stats && d_dlogits, "cfp_token_logprobs_grad: NULL stats or output");
    CFP_REQUIRE(top == 0 || (d_top_ids && d_g_top), "cfp_token_logprobs_grad: top = %d needs the ids and their gradients", top);
    CFP_REQUIRE(ld_dlogits >= vocab || (rows == 1 && ld_dlogits >= 0), "cfp_token_logprobs_grad: rows of %d gradients need a stride of at least that (got %lld)",
                vocab, (long long)ld_dlogits);
    CFP_REQUIRE((reinterpret_cast<uintptr_t>(d_dlogits) & (dtype == CFP_F32 ? 3u : 1u)) == 0,
                "cfp_token_logprobs_grad: output not aligned to its type");
    const char *x0 = (const char*)d_logits, *y0 = (const char*)d_dlogits;
    const char* x1 = x0 + ((size_t)(rows - 1) * ld + vocab) * elem_bytes(dtype);
    const char* y1 = y0 + ((size_t)(rows - 1) * ld_dlogits + vocab) * elem_bytes(dtype);
    CFP_REQUIRE(y0 >= x1 || x0 >= y1 || (x0 == y0 && (ld == ld_dlogits || rows == 1)),
                "cfp_token_logprobs_grad: the gradient may replace the logits, with the same stride, but not overlap them otherwise");
    const LpPlan pl = plan_grad(rows, vocab);
    CFP_REQUIRE(pl.kind < 2 || (int64_t)rows * pl.splits <= kMaxGroups, "cfp_token_logprobs_grad: %d rows of %d are more than one launch holds",
                rows, vocab);
    LpGradArgs a{};
    a.x = d_logits; a.ld = ld; a.rows = rows; a.vocab = vocab; a.tok = d_tokens;
    a.mask = d_mask; a.ld_mask = ld_mask; a.stats = d_stats;
    a.g_lp = d_g_logprobs; a.g_ent = d_g_entropy; a.top = top; a.ids = d_top_ids; a.g_top = d_g_top;
    a.dx = d_dlogits; a.ld_dx = ld_dlogits; a.splits = pl.splits; a.chunk = pl.chunk;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == CFP_F32) { d_mask ? run_grad<float, true>(a, pl, st) : run_grad<float, false>(a, pl, st); }
    else if (dtype == CFP_BF16) { d_mask ? run_grad<__bf16, true>(a, pl, st) : run_grad<__bf16, false>(a, pl, st); }
    else { d_mask ? run_grad<_Float16, true>(a, pl, st) : run_grad<_Float16, false>(a, pl, st); }
    CFP_HIP_TRY(hipGetLastError());
    return 0;
}

}  // extern "C"
