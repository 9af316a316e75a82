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
// m + ln s has lost the bits of ln s.  All sums are fp32 per lane, of 512 terms in [0, 1] and the
// entries of one more tile at most (rows above 2^17 entries are split for it), and joined in a tree of
// fixed shape: the same call gives the same bits.
#include <float.h>
#include <limits.h>

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
// All-reduce over 16 or 64 consecutive lanes in a tree of fixed shape.  Rotations inside rows of
// 16 lanes ride on the addition itself (a shuffle through LDS a step instead: 27 us for 262 144
// rows of 43 where this takes 20).
template <int D>
__device__ __forceinline__ unsigned xor_lane(unsigned v) {
    if (D == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);     // within quads
    if (D == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);
    if (D == 4)   // mirrored in eights, then in quads
        return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true), 0x1b, 0xf, 0xf, true);
    if (D == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);    // rotated by half a row
    if (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
}
template <int N>
__device__ __forceinline__ float row_rotate(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + N, 0xf, 0xf, true));
}
template <int WIDTH, class Op>
__device__ __forceinline__ float reduce_lanes(float v, Op op) {
    static_assert(WIDTH == 16 || WIDTH == 64, "rows of 16 lanes or the wavefront");
    v = op(v, row_rotate<8>(v));
    v = op(v, row_rotate<4>(v));
    v = op(v, row_rotate<2>(v));
    v = op(v, row_rotate<1>(v));
    if (WIDTH == 64) {
        v = op(v, __uint_as_float(xor_lane<16>(__float_as_uint(v))));
        v = op(v, __uint_as_float(xor_lane<32>(__float_as_uint(v))));
    }
    return v;
}
template <int WIDTH>
__device__ __forceinline__ float sum_lanes(float v) {
    return reduce_lanes<WIDTH>(v, [](float a, float b) { return a + b; });
}
template <int WIDTH>
__device__ __forceinline__ float max_lanes(float v) {
    return reduce_lanes<WIDTH>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int WIDTH>
__device__ __forceinline__ int min_lanes(int v) {
    v = min(v, (int)xor_lane<1>((unsigned)v));
    v = min(v, (int)xor_lane<2>((unsigned)v));
    v = min(v, (int)xor_lane<4>((unsigned)v));
    v = min(v, (int)xor_lane<8>((unsigned)v));
    if (WIDTH == 64) {
        v = min(v, (int)xor_lane<16>((unsigned)v));
        v = min(v, (int)xor_lane<32>((unsigned)v));
    }
    return v;
}
__device__ __forceinline__ void join_lanes(Sums& a) {
    raise_max(a, max_lanes<64>(a.m));
    a.s = sum_lanes<64>(a.s);
    a.u = sum_lanes<64>(a.u);
}

// ---- the best `top` entries seen by one wavefront -----------------------------------
// An entry is one 64-bit key, larger = better: the value's bits in unsigned order (0 and -0 the
// same), then the complement of the index, so that equal values go to the lower index.  0 is a
// free place; NaN and -inf never become keys.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    const unsigned u = __float_as_uint(v + 0.0f);
    return (uint64_t)(u ^ ((unsigned)((int)u >> 31) | 0x80000000u)) << 32 | (unsigned)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const unsigned h = (unsigned)(k >> 32);
    return k == 0 ? -INFINITY : __uint_as_float(h & 0x80000000u ? h ^ 0x80000000u : ~h);
}
__device__ __forceinline__ int key_index(uint64_t k) { return ~(int)(unsigned)k; }
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane) {
    return (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)k, lane);
}
template <int D>
__device__ __forceinline__ uint64_t xor_key(uint64_t k) {
    return (uint64_t)xor_lane<D>((unsigned)(k >> 32)) << 32 | xor_lane<D>((unsigned)k);
}
// runs of 2 D become sorted, best first where `best_first` (alternating by bit 2 D of the lane),
// from runs of D that alternate
template <int STEP>
__device__ __forceinline__ void merge_runs(uint64_t& k, bool best_first) {
    const uint64_t other = xor_key<STEP>(k);
    const bool keep_better = ((threadIdx.x & STEP) == 0) == best_first;
    if ((other > k) == keep_better) k = other;
    if constexpr (STEP > 1) merge_runs<STEP / 2>(k, best_first);
}
// Lane i of `key` holds the entry of rank i.  An entry that beats the one of rank top - 1 goes to
// a buffer in LDS; when that holds 64, they are sorted across the lanes (21 exchanges) and merged
// with the list (6).  On values in random order the bar rises fast enough for the merges to
// number about log4(entries / 64); one insertion at a time, about top * ln(entries / top) of
// them and each as long as a few exchanges, took 34 us for 1 x 131 072 where this takes 9.
constexpr int kBuffer = 128;   // of which 64 trigger a merge
struct Best {
    uint64_t key = 0;
    uint64_t last = 0;          // the entry of rank top - 1: what a newcomer has to beat
    float last_v = -INFINITY;   // its value
    int waiting = 0;            // entries in the buffer; wave-uniform
    uint64_t* buffer;           // [kBuffer] of this wavefront

    __device__ __forceinline__ static void sort(uint64_t& k, bool best_first) {
        const int lane = threadIdx.x & 63;
        merge_runs<1>(k, (lane & 2) == 0);
        merge_runs<2>(k, (lane & 4) == 0);
        merge_runs<4>(k, (lane & 8) == 0);
        merge_runs<8>(k, (lane & 16) == 0);
        merge_runs<16>(k, (lane & 32) == 0);
        merge_runs<32>(k, best_first);
    }
    // A bar for an empty list: every lane names the largest of the entries that it is about to
    // offer, and what does not reach the top-th largest of those cannot be among the best.  Of a
    // first tile about 1.2 top entries remain.
    __device__ __forceinline__ void set_bar(float largest, int top) {
        if (last != 0) return;
        if (top <= 8) {   // maxima one by one: 12 instructions each, the sort 190
            float v = largest;
            for (int k = 0; k < top; k++) {
                last_v = max_lanes<64>(v);
                const unsigned long long who = __ballot(v == last_v);
                if ((int)(threadIdx.x & 63) == __ffsll(who) - 1) v = -INFINITY;
            }
            last = last_v > -INFINITY ? key_of(last_v, -1) : 0;   // index -1: entries equal to the bar pass
            return;
        }
        uint64_t k = largest > -INFINITY ? key_of(largest, -1) : 0;
        sort(k, true);
        last = lane_key(k, top - 1);
        last_v = key_value(last);
    }
    // the first 64 of the buffer into the list
    __device__ __forceinline__ void merge(int top) {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint64_t c = lane < waiting ? buffer[lane] : 0;
        if (waiting > 64) {   // the rest moves to the front
            const uint64_t rest = buffer[64 + lane];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            buffer[lane] = rest;
        }
        waiting = waiting > 64 ? waiting - 64 : 0;
        sort(c, false);   // worst first: against the list it makes one bitonic run
        if (c > key) key = c;
        merge_runs<32>(key, true);
        const uint64_t bar = lane_key(key, top - 1);
        if (bar > last) { last = bar; last_v = key_value(bar); }
    }
    // one entry a lane (wave-uniform call)
    __device__ __forceinline__ void offer(float x, int idx, int top) { offer(x > -INFINITY ? key_of(x, idx) : 0, top); }
    __device__ __forceinline__ void offer(uint64_t k, int top) {
        const bool mine = k > last;
        const unsigned long long who = __ballot(mine);
        if (who == 0) return;
        if (mine) buffer[waiting + __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0))] = k;
        waiting += __popcll(who);
        if (waiting >= 64) merge(top);
    }
    __device__ __forceinline__ void finish(int top) {
        if (waiting > 0) merge(top);
    }
};

// the same for 16-bit types and indices below 2^16
template <typename T>
__device__ __forceinline__ unsigned short_key(float v, int i) {
    const unsigned u = __builtin_bit_cast(unsigned short, (T)(v + 0.0f));   // exact: v came from a T
    return (u ^ (u & 0x8000u ? 0xffffu : 0x8000u)) << 16 | (unsigned)(0xffff - i);
}
template <typename T>
__device__ __forceinline__ float short_value(unsigned key) {
    const unsigned h = key >> 16;
    return to_f32(__builtin_bit_cast(T, (unsigned short)(h & 0x8000u ? h ^ 0x8000u : h ^ 0xffffu)));
}

struct LpArgs {
    const void* x;
    int64_t ld;
    int rows, vocab;
    const int32_t* tok;
    const uint8_t* mask;   // or null
    int64_t ld_mask;       // 0: one mask for all rows
    float* lp;
    float* ent;            // or null
    int row0;              // of this launch (k_logprobs_short)
    int top;
    int32_t* ids;
    float* top_lp;
    float* stats;          // [rows][3] or null
    int splits, chunk;     // entries per split, a multiple of 8
    f4* part;              // [rows][splits] (m, s, u, -)
    uint64_t* part_top;    // [rows][splits][top] keys
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
__device__ __forceinline__ void write_top(const LpArgs& a, int row, const Sums& z, int rank, uint64_t key) {
    const float v = key_value(key);
    const int i = key_index(key);
    const size_t o = (size_t)row * a.top + rank;
    const bool bad = z.s != z.s;   // NaN or +inf among the allowed entries
    a.ids[o] = bad ? -1 : i;   // a free place has index -1
    a.top_lp[o] = bad ? NAN : key == 0 ? -INFINITY : (v - z.m) - logf(z.s);
}
template <typename T>
__device__ __forceinline__ float token_logit(const LpArgs& a, int row, int tok) {
    if (tok < 0 || tok >= a.vocab) return -INFINITY;
    const float x = to_f32(((const T*)a.x)[(size_t)row * a.ld + tok]);
    if (a.mask && a.mask[(size_t)row * a.ld_mask + tok] == 0) return -INFINITY;
    return x;
}

// ---- short rows: L lanes a row, Q 16-byte vectors a lane ----------------------------------
// The row sits in registers: the maximum first, then the exponentials, no rescaling.  The last
// vector of a row is moved back to end with it; the entries it shares with the one before count
// once (as -inf here).
constexpr int kShortBytes = 2048;   // of a row: 64 lanes, two vectors each
template <typename T, int L, int Q, bool MASK>
__device__ __forceinline__ void load_short(const T* x, const uint8_t* mask, int vocab, int sub, float (&v)[Q][Vec<T>::N],
                                           int (&first)[Q]) {
    constexpr int N = Vec<T>::N;
    if (vocab < N) {   // not even one vector
#pragma unroll
        for (int q = 0; q < Q; q++) {
            first[q] = q == 0 && sub == 0 ? 0 : vocab;
#pragma unroll
            for (int j = 0; j < N; j++) {
                v[q][j] = -INFINITY;
                if (first[q] + j < vocab && (!MASK || mask[j])) v[q][j] = to_f32(x[j]);
            }
        }
        return;
    }
    Vec<T> raw[Q];
    uint8_t mk[Q][N];
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const int i = (q * L + sub) * N;
        first[q] = min(i, vocab - N);
        raw[q] = load_vec(x + first[q]);   // lanes behind the row repeat its last vector
        if (MASK) __builtin_memcpy(mk[q], mask + first[q], N);
    }
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const int i = (q * L + sub) * N;
#pragma unroll
        for (int j = 0; j < N; j++)
            v[q][j] = first[q] + j < i || (MASK && mk[q][j] == 0) ? -INFINITY : to_f32(raw[q].v[j]);
    }
}
template <typename T, int L, int Q, bool MASK>
__global__ __launch_bounds__(256) void k_logprobs_short(LpArgs a) {
    constexpr int N = Vec<T>::N;
    const int sub = threadIdx.x % L;
    const unsigned row = (unsigned)a.row0 + blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = row < (unsigned)a.rows;
    const int r = live ? (int)row : a.rows - 1;
    const int tok = a.tok[r];
    const float xt = token_logit<T>(a, r, tok);
    float v[Q][N];
    int first[Q];
    load_short<T, L, Q, MASK>((const T*)a.x + (size_t)r * a.ld, MASK ? a.mask + (size_t)r * a.ld_mask : nullptr,
                              a.vocab, sub, v, first);
    Sums z;
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
        for (int j = 0; j < N; j++) z.m = fmaxf(z.m, v[q][j]);
    z.m = max_lanes<L>(z.m);
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
        for (int j = 0; j < N; j++) add_entry(z, v[q][j]);
    z.s = sum_lanes<L>(z.s);
    z.u = sum_lanes<L>(z.u);
    if (live && sub == 0) write_row(a, r, z, tok, xt);
    if (a.top == 0) return;
    // Alternatives: the maximum of the row, then the lowest index that holds it, `top` times; lane
    // k (then k - L) keeps number k, and all are written together.  16-bit entries and their index
    // make one 32-bit key (rows have at most 1024 of them): 262 144 x 43 fp16 with 20 alternatives
    // take 85 us, 150 with value and index apart, as fp32 has them (111).
    constexpr int SLOTS = kMaxTop > L ? kMaxTop / L : 1;
    if constexpr (sizeof(T) == 2) {
        unsigned key[Q][N], kept[SLOTS] = {};
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int j = 0; j < N; j++) key[q][j] = v[q][j] > -INFINITY ? short_key<T>(v[q][j], first[q] + j) : 0u;
        for (int k = 0; k < a.top; k++) {   // wave-uniform trip count
            unsigned best = 0;
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int j = 0; j < N; j++) best = max(best, key[q][j]);
            best = max(best, xor_lane<1>(best));
            best = max(best, xor_lane<2>(best));
            best = max(best, xor_lane<4>(best));
            best = max(best, xor_lane<8>(best));
            if (L == 64) {
                best = max(best, xor_lane<16>(best));
                best = max(best, xor_lane<32>(best));
            }
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int j = 0; j < N; j++) key[q][j] = key[q][j] == best ? 0u : key[q][j];
#pragma unroll
            for (int t = 0; t < SLOTS; t++) kept[t] = k == t * L + sub ? best : kept[t];
        }
#pragma unroll
        for (int t = 0; t < SLOTS; t++)
            if (live && t * L + sub < a.top)
                write_top(a, r, z, t * L + sub, kept[t] ? key_of(short_value<T>(kept[t]), 0xffff - (int)(kept[t] & 0xffffu)) : 0);
        return;
    }
    uint64_t kept[SLOTS] = {};
    for (int k = 0; k < a.top; k++) {   // wave-uniform trip count
        float bv = -INFINITY;
        int bi = INT_MAX;
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int j = 0; j < N; j++)   // ascending index: ties keep the first
                if (v[q][j] > bv) { bv = v[q][j]; bi = first[q] + j; }
        const float m = max_lanes<L>(bv);
        bi = min_lanes<L>(bv == m ? bi : INT_MAX);
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int j = 0; j < N; j++)
                if (first[q] + j == bi) v[q][j] = -INFINITY;
#pragma unroll
        for (int t = 0; t < SLOTS; t++)
            if (k == t * L + sub) kept[t] = bi == INT_MAX ? 0 : key_of(m, bi);
    }
#pragma unroll
    for (int t = 0; t < SLOTS; t++)
        if (live && t * L + sub < a.top) write_top(a, r, z, t * L + sub, kept[t]);
}

// ---- short rows, many of them: one thread a row ------------------------------------------
// The lanes of the kernel above spend 37 instructions a row (reductions, addresses, logarithm, each
// on all 16 lanes); with rows staged through LDS and one thread a row it is about 8, and the
// kernel is bound by HBM.  Fewer rows leave the machine idle this way: from kRowsFrom on.
// The rows of LDS are an odd number of floats apart, so the threads' rows start in different banks.
// Rows travel as 16-byte vectors whatever their alignment; the last vector of a row is moved back
// to end with it, so it overlaps the one before (whose entries it repeats).
constexpr int kRowsMax = 64, kRowsThreads = 128, kRowsFrom = 16384;
__host__ __device__ inline int rows_pitch(int vocab) { return vocab | 1; }
// vector q of kRowsThreads rows of `vocab` entries: its row and first entry
template <int N>
struct RowVectors {
    int vocab, per_row;
    unsigned inv;
    __device__ __forceinline__ explicit RowVectors(int v) : vocab(v), per_row((v + N - 1) / N) {
        inv = ((1u << 20) + per_row - 1) / per_row;   // q / per_row = q * inv / 2^20 for q < 2^11
    }
    __device__ __forceinline__ void at(int q, int& row, int& first) const {
        row = (int)(((unsigned)q * inv) >> 20);
        first = min((q - row * per_row) * N, vocab - N);
    }
};
// `rows` rows from x on (kRowsThreads at most) as fp32 into LDS, -inf where masked; all of a thread's
// loads in flight together (at most PASSES; per_row of them).
template <typename T, int PASSES, bool MASK>
__device__ __forceinline__ void stage_rows(const T* x, int64_t ld, const uint8_t* mask, int64_t ld_mask, int rows, int vocab,
                                           float* stage) {
    constexpr int N = Vec<T>::N;
    const RowVectors<N> rv(vocab);
    Vec<T> v[PASSES];
    uint8_t mk[PASSES][N];
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        int r, i;
        rv.at(p * kRowsThreads + (int)threadIdx.x, r, i);
        if (p >= rv.per_row || r >= rows) continue;
        v[p] = load_vec(x + (size_t)r * ld + i);
        if (MASK) __builtin_memcpy(mk[p], mask + (size_t)r * ld_mask + i, N);
    }
    const int pitch = rows_pitch(vocab);
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        int r, i;
        rv.at(p * kRowsThreads + (int)threadIdx.x, r, i);
        if (p >= rv.per_row || r >= rows) continue;
#pragma unroll
        for (int j = 0; j < N; j++) stage[r * pitch + i + j] = MASK && mk[p][j] == 0 ? -INFINITY : to_f32(v[p].v[j]);
    }
}
template <typename T, int PASSES, bool MASK>
__global__ __launch_bounds__(kRowsThreads) void k_logprobs_rows(LpArgs a) {
    extern __shared__ float stage[];
    const int r0 = (int)blockIdx.x * kRowsThreads, row = r0 + (int)threadIdx.x, here = min(kRowsThreads, a.rows - r0);
    const bool live = row < a.rows;
    stage_rows<T, PASSES, MASK>((const T*)a.x + r0 * a.ld, a.ld, MASK ? a.mask + r0 * a.ld_mask : nullptr, a.ld_mask, here,
                                a.vocab, stage);
    const int tok = live ? a.tok[row] : -1;
    __syncthreads();
    if (live) {
        const float* x = stage + threadIdx.x * rows_pitch(a.vocab);
        Sums z;
#pragma unroll 4
        for (int i = 0; i < a.vocab; i++) z.m = fmaxf(z.m, x[i]);
#pragma unroll 4
        for (int i = 0; i < a.vocab; i++) add_entry(z, x[i]);
        write_row(a, row, z, tok, tok >= 0 && tok < a.vocab ? x[tok] : -INFINITY);
    }
}

// ---- long rows -------------------------------------------------------------------------
// One tile: kU vectors a lane, all loads in flight before the first use.
constexpr int kU = 4;
// Candidates of a tile: lanes that hold one put their 64 bytes of it into LDS (raw type, masked
// entries as -inf), rows kLaneBytes apart, and the wavefront offers one or a few such lanes'
// entries at a time.  (Offering the 32 registers in turn is 32 copies of the merge: 298 us for
// 4096 x 131 072 instead of 195.)
constexpr int kLaneBytes = 80;
struct TopSpace {
    uint64_t buffer[kBuffer];
    __align__(16) unsigned char tile[64 * kLaneBytes];
};
template <typename T>
__device__ __forceinline__ void offer_tile(const float (&v)[kU][Vec<T>::N], float tm, int base, int stride, int lane0,
                                           unsigned char* tile, Best& best, int top) {
    constexpr int N = Vec<T>::N, PER = kU * N, TOGETHER = 64 / PER;
    const int lane = threadIdx.x & 63;
    best.set_bar(tm, top);
    const bool mine = tm >= best.last_v && tm > -INFINITY;
    unsigned long long todo = __ballot(mine);
    if (todo == 0) return;
    if (mine)
#pragma unroll
        for (int q = 0; q < kU; q++) {
            Vec<T> raw;
#pragma unroll
            for (int j = 0; j < N; j++) raw.v[j] = (T)v[q][j];   // exact: it came from a T
            *reinterpret_cast<u4*>(tile + lane * kLaneBytes + 16 * q) = __builtin_bit_cast(u4, raw);
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int slot = lane % PER, q = slot / N, j = slot % N;
    while (todo) {
        int src = -1;
#pragma unroll
        for (int k = 0; k < TOGETHER; k++) {
            if (todo && lane / PER == k) src = __ffsll((long long)todo) - 1;
            todo &= todo - 1;   // 0 stays 0
        }
        float x = -INFINITY;
        if (src >= 0) x = to_f32(*reinterpret_cast<const T*>(tile + src * kLaneBytes + 16 * q + j * (int)sizeof(T)));
        best.offer(x, base + q * stride + (lane0 + src) * N + j, top);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// W wavefronts of a workgroup stream entries [lo, hi) of a row; thread t takes vectors t,
// t + 64 W, ...  Every wavefront runs the same number of tiles (uniform trip count).
template <typename T, bool MASK, bool TOP, int W>
__device__ __forceinline__ void stream_row(const T* x, const uint8_t* mask, int lo, int hi, Sums& z, Best& best,
                                           TopSpace* space, int top) {
    constexpr int N = Vec<T>::N, STRIDE = 64 * W * N, TILE = STRIDE * kU;
    const int t = W == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    for (int base = lo; base < hi; base += TILE) {
        const int i0 = base + t * N;
        float v[kU][N];
        if (base + TILE <= hi) {
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
                for (int j = 0; j < N; j++) v[q][j] = MASK && mk[q][j] == 0 ? -INFINITY : to_f32(raw[q].v[j]);
        } else {   // the last, partial tile: whole vectors where they fit, entries at the end
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
        }
        float tm = v[0][0];
#pragma unroll
        for (int q = 0; q < kU; q++)
            if (q == 0 || base + q * STRIDE < hi)   // a partial tile has fewer
#pragma unroll
                for (int j = 0; j < N; j++) tm = fmaxf(tm, v[q][j]);
        if (tm > z.m) raise_max(z, tm);
#pragma unroll
        for (int q = 0; q < kU; q++)
            if (q == 0 || base + q * STRIDE < hi)
#pragma unroll
                for (int j = 0; j < N; j++) add_entry(z, v[q][j]);
        if (TOP) offer_tile<T>(v, tm, base, STRIDE, t - (int)(threadIdx.x & 63), space->tile, best, top);
    }
}

// One wavefront a row, four rows a workgroup: rows that are many or not long.
template <typename T, bool MASK, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_wave(LpArgs a) {
    __shared__ TopSpace spaces[TOP ? 4 : 1];
    const int lane = threadIdx.x & 63;
    for (int64_t row0 = (int64_t)blockIdx.x * 4; row0 < a.rows; row0 += (int64_t)gridDim.x * 4) {
        if (row0 + (threadIdx.x >> 6) >= a.rows) return;   // whole wavefronts; nothing below synchronises a workgroup
        const int row = (int)row0 + (int)(threadIdx.x >> 6);
        const int tok = a.tok[row];
        const float xt = token_logit<T>(a, row, tok);
        Sums z;
        Best best;
        TopSpace* space = &spaces[TOP ? threadIdx.x >> 6 : 0];
        best.buffer = space->buffer;
        stream_row<T, MASK, TOP, 1>((const T*)a.x + (size_t)row * a.ld,
                                    MASK ? a.mask + (size_t)row * a.ld_mask : nullptr, 0, a.vocab, z, best, space,
                                    a.top);
        join_lanes(z);
        if (lane == 0) write_row(a, row, z, tok, xt);
        if (TOP) best.finish(a.top);
        if (TOP && lane < a.top) write_top(a, row, z, lane, best.key);
    }
}

// One workgroup for entries [split * chunk, ...) of a row; with one split it writes the
// outputs, else its part, which k_logprobs_join puts together.
constexpr int kWaves = 4;
template <typename T, bool MASK, bool TOP>
__global__ __launch_bounds__(64 * kWaves) void k_logprobs_group(LpArgs a) {
    __shared__ float zs[kWaves][3];
    __shared__ TopSpace spaces[TOP ? kWaves : 1];
    __shared__ uint64_t lists[TOP ? kWaves : 1][kMaxTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
    const int lo = split * a.chunk, hi = lo + a.chunk < a.vocab ? lo + a.chunk : a.vocab;
    const int tok = a.tok[row];
    const float xt = a.splits == 1 ? token_logit<T>(a, row, tok) : 0.0f;
    Sums z;
    Best best;
    TopSpace* space = &spaces[TOP ? wave : 0];
    best.buffer = space->buffer;
    stream_row<T, MASK, TOP, kWaves>((const T*)a.x + (size_t)row * a.ld,
                                     MASK ? a.mask + (size_t)row * a.ld_mask : nullptr, lo, hi, z, best, space, a.top);
    join_lanes(z);
    if (lane == 0) { zs[wave][0] = z.m; zs[wave][1] = z.s; zs[wave][2] = z.u; }
    if (TOP) best.finish(a.top);
    if (TOP && wave > 0 && lane < a.top) lists[wave][lane] = best.key;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; w++) join(z, zs[w][0], zs[w][1], zs[w][2]);
    if (TOP) {
        for (int w = 1; w < kWaves; w++) best.offer(lane < a.top ? lists[w][lane] : 0, a.top);
        best.finish(a.top);
    }
    if (a.splits == 1) {
        if (lane == 0) write_row(a, row, z, tok, xt);
        if (TOP && lane < a.top) write_top(a, row, z, lane, best.key);
        return;
    }
    const size_t o = (size_t)row * a.splits + split;
    if (lane == 0) a.part[o] = f4{z.m, z.s, z.u, 0.0f};
    if (TOP && lane < a.top) a.part_top[o * a.top + lane] = best.key;
}

// One wavefront a row: the parts of its splits in ascending order of lane, then the tree.
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_join(LpArgs a) {
    __shared__ uint64_t buffer[kBuffer];
    const int lane = threadIdx.x, row = (int)blockIdx.x;
    const int tok = a.tok[row];
    const float xt = token_logit<T>(a, row, tok);
    Sums z;
    for (int s = lane; s < a.splits; s += 64) {
        const f4 p = a.part[(size_t)row * a.splits + s];
        join(z, p[0], p[1], p[2]);
    }
    join_lanes(z);
    if (lane == 0) write_row(a, row, z, tok, xt);
    if (a.top > 0) {
        Best best;
        best.buffer = buffer;
        const int total = a.splits * a.top;
        const uint64_t* keys = a.part_top + (size_t)row * total;
        best.set_bar(lane < a.splits ? key_value(keys[lane * a.top]) : -INFINITY, a.top);
        for (int o = 0; o < total; o += 64) best.offer(o + lane < total ? keys[o + lane] : 0, a.top);
        best.finish(a.top);
        if (lane < a.top) write_top(a, row, z, lane, best.key);
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
    int row0;              // of this launch (k_logprobs_grad_short, k_logprobs_grad)
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
template <typename T, int L, int Q, bool MASK>
__global__ __launch_bounds__(256) void k_logprobs_grad_short(LpGradArgs a) {
    constexpr int N = Vec<T>::N;
    const int sub = threadIdx.x % L;
    const unsigned row = (unsigned)a.row0 + blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = row < (unsigned)a.rows;
    const int r = live ? (int)row : a.rows - 1;
    float v[Q][N], d[Q][N];
    int first[Q];
    load_short<T, L, Q, MASK>((const T*)a.x + (size_t)r * a.ld, MASK ? a.mask + (size_t)r * a.ld_mask : nullptr,
                              a.vocab, sub, v, first);
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
        for (int j = 0; j < N; j++) d[q][j] = 0.0f;
    // the named entries: whose lane holds an allowed one takes its gradient
    float weight = 0.0f;
    for (int k = 0; k <= a.top; k++) {
        if (k == 0 && !a.g_lp) continue;
        const int i = k == 0 ? a.tok[r] : a.ids[(size_t)r * a.top + k - 1];
        const float g = k == 0 ? a.g_lp[r] : a.g_top[(size_t)r * a.top + k - 1];
        if (i >= a.vocab && sub == 0) weight = NAN;
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int j = 0; j < N; j++)
                if (first[q] + j == i && !(v[q][j] == -INFINITY)) { d[q][j] += g; weight += g; }
    }
    RowGrad rg;
    row_grad(a, r, sum_lanes<L>(weight), rg);
    T* dx = (T*)a.dx + (size_t)r * a.ld_dx;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        // every load of this row was used above: the row may be overwritten in place.  Each
        // entry is stored by the lane that it counts for.
        const int i = (q * L + sub) * N;
        Vec<T> out;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const bool on = !rg.none && !(v[q][j] == -INFINITY);
            out.v[j] = (T)(on ? rg.at(v[q][j]) + d[q][j] : 0.0f);
        }
        if (!live) continue;
        if (i + N <= a.vocab) store_vec(dx + i, out);
        else
#pragma unroll
            for (int j = 0; j < N; j++)
                if (first[q] + j >= i && first[q] + j < a.vocab) dx[first[q] + j] = out.v[j];
    }
}

// one thread a row, as k_logprobs_rows; the gradient replaces the logits in LDS
template <typename T, int PASSES, bool MASK>
__global__ __launch_bounds__(kRowsThreads) void k_logprobs_grad_rows(LpGradArgs a) {
    extern __shared__ float stage[];
    constexpr int N = Vec<T>::N;
    const int pitch = rows_pitch(a.vocab);
    const int r0 = (int)blockIdx.x * kRowsThreads, row = r0 + (int)threadIdx.x, here = min(kRowsThreads, a.rows - r0);
    const bool live = row < a.rows;
    stage_rows<T, PASSES, MASK>((const T*)a.x + r0 * a.ld, a.ld, MASK ? a.mask + r0 * a.ld_mask : nullptr, a.ld_mask, here,
                                a.vocab, stage);
    int tok = -1;
    float g = 0.0f;
    if (live && a.g_lp) { tok = a.tok[row]; g = a.g_lp[row]; }
    __syncthreads();
    if (live) {
        float* x = stage + threadIdx.x * pitch;
        const bool hit = tok >= 0 && tok < a.vocab && !(x[tok] == -INFINITY);
        RowGrad rg;
        row_grad(a, row, tok >= a.vocab ? NAN : hit ? g : 0.0f, rg);
#pragma unroll 4
        for (int i = 0; i < a.vocab; i++) {
            const float v = x[i];
            x[i] = rg.none || v == -INFINITY ? 0.0f : rg.at(v) + (i == tok ? g : 0.0f);
        }
    }
    __syncthreads();
    T* dx = (T*)a.dx + r0 * a.ld_dx;
    if (a.ld_dx == a.vocab && pitch == a.vocab && here * pitch % N == 0 && (reinterpret_cast<uintptr_t>(a.dx) & 15u) == 0) {
        // rows without gaps, in memory and (odd widths) in LDS: one run of aligned vectors (r0 is a
        // multiple of kRowsThreads)
#pragma unroll 4
        for (int e = (int)threadIdx.x * N; e < here * pitch; e += kRowsThreads * N) {
            Vec<T> out;
#pragma unroll
            for (int j = 0; j < N; j++) out.v[j] = (T)stage[e + j];
            store_vec(dx + e, out);
        }
    } else {
        const RowVectors<N> rv(a.vocab);
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            int r, i;
            rv.at(p * kRowsThreads + (int)threadIdx.x, r, i);
            if (p >= rv.per_row || r >= here) continue;
            Vec<T> out;
#pragma unroll
            for (int j = 0; j < N; j++) out.v[j] = (T)stage[r * pitch + i + j];
            store_vec(dx + (size_t)r * a.ld_dx + i, out);   // repeated entries: the same values
        }
    }
}

// Entries [lo, hi) of a row by one workgroup: what all entries have in common first, then the
// named entries (given token, alternatives) once more by one lane each.  Their logits are read
// before the first store, their values stored behind the last one (barriers on both sides).  The
// barriers order one workgroup only, and every workgroup of a row reads all of its named logits:
// where dx is x, a row has one workgroup (plan_grad), of kInPlaceThreads (bf16, in parts to another
// array / in place by 256 / 512 / 1024 threads: 1 x 131 072 4 / 27 / 17 / 15 us, 128 x 131 072
// 15 / 33 / 22 / 20, 2048 x 131 072 195 / 217 / 209 / 196, 4096 x 50 021 206 / 176 / 171 / 217,
// 4096 x 4000 32 / 22 / 26 / 32).
constexpr int kInPlaceThreads = 512;
template <typename T, bool MASK, int THREADS>
__global__ __launch_bounds__(THREADS) void k_logprobs_grad(LpGradArgs a) {
    constexpr int N = Vec<T>::N, STRIDE = THREADS * N, TILE = STRIDE * kU;
    const int row = a.row0 + (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
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
    for (int i = base + (int)threadIdx.x; i < hi; i += THREADS) {
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
// Rows of up to 2 KiB sit in the registers of 16 or 64 lanes (1 KiB from four alternatives on in
// fp32, 512 bytes from nine on: finding them one by one costs 30 to 110 instructions each there,
// sorting candidates about 500 once; 100 000 x 300 fp32 with 5: 99 us against 125, 41 943 x 800 fp16
// with 5: 46 against 55, 83 886 x 400 fp16 with 32: 173 against 139).  Longer ones are streamed: by
// a wavefront each where there are enough rows to fill the machine that way (256 CUs, 16
// wavefronts each) and a row is not so long that its last wavefronts run alone; by a workgroup
// each otherwise, split further until about four workgroups a CU run, none with less than 4096
// entries (one tile of 16-bit loads is 8192, and a second launch joins the parts).  Parts hold at most
// kMostEntries, 512 a lane: roundings of a longer running sum of equal terms all go one way (2.3e-4 of
// the sum after 16 384 terms).
constexpr int kMostEntries = 512 * 64 * kWaves;
LpPlan plan_forward(int rows, int vocab, int bytes, int top) {
    const int whole = bytes == 2 ? 8 : 3;   // alternatives for which a row may have all of kShortBytes
    if ((int64_t)vocab * bytes <= (top <= whole ? kShortBytes : top <= 8 ? kShortBytes / 2 : kShortBytes / 4)) return {0, 1, 0};
    if (rows >= 4096 && vocab <= 8192) return {1, 1, 0};
    const int want = rows >= 512 ? 1 : (1024 + rows - 1) / rows;
    const int most = (vocab + 4095) / 4096, least = (vocab + kMostEntries - 1) / kMostEntries;
    int splits = want < least ? least : want < most ? want : most;
    const int chunk = ((vocab + splits - 1) / splits + 7) / 8 * 8;
    splits = (vocab + chunk - 1) / chunk;
    return {2, splits, chunk};
}
// the gradient's parts are independent unless it replaces the logits: 16384 entries a workgroup at
// most, 1024 at least
LpPlan plan_grad(int rows, int vocab, int bytes, bool in_place) {
    if ((int64_t)vocab * bytes <= kShortBytes) return {0, 1, 0};
    if (in_place) return {2, 1, vocab};
    int splits = (vocab + 16383) / 16384;
    while ((int64_t)rows * splits < 2048 && (vocab + splits - 1) / splits > 2048) splits *= 2;
    const int chunk = ((vocab + splits - 1) / splits + 7) / 8 * 8;
    return {2, (vocab + chunk - 1) / chunk, chunk};
}
size_t part_bytes(int rows, int splits, int top) {
    return splits == 1 ? 0 : (size_t)rows * splits * (sizeof(f4) + (size_t)top * sizeof(uint64_t));
}

constexpr int kMaxVocab = 1 << 30;
// workgroups of a launch: threads of a grid are counted in 32 bits
constexpr int64_t kMaxGroups = ((int64_t)1 << 32) / 256 - 1;
int capped_groups(int64_t g) { return (int)(g < kMaxGroups ? g : kMaxGroups); }

// one thread a row has no use for alternatives: 16 lanes find them together
// (8: a vector of 16-bit logits)
bool by_rows(int rows, int vocab, int top) { return rows >= kRowsFrom && vocab >= 8 && vocab <= kRowsMax && top == 0; }
int rows_groups(int rows) { return (int)(((int64_t)rows + kRowsThreads - 1) / kRowsThreads); }   // at most 2^31 threads
size_t rows_lds(int vocab) { return (size_t)kRowsThreads * rows_pitch(vocab) * sizeof(float); }

// launch(arguments, grid) for all rows, `per` of them a workgroup and as many a launch as it has
// workgroups for.  (Loops over rows inside the kernels, in 64 bits, cost registers and instructions:
// scores of 100 000 x 300 fp32 46 us instead of 38, the gradient of 1001 x 32 003 fp16 with a mask 47
// instead of 38.)
template <class Args, class Launch>
void in_launches(Args a, int64_t per, Launch launch) {
    const int64_t most = kMaxGroups * per;
    for (int64_t row0 = 0; row0 < a.rows; row0 += most) {
        const int64_t here = a.rows - row0 < most ? a.rows - row0 : most;
        a.row0 = (int)row0;
        launch(a, dim3((unsigned)((here + per - 1) / per)));
    }
}

template <typename T, bool MASK>
void run_forward(const LpArgs& a, const LpPlan& pl, hipStream_t st) {
    if (pl.kind == 0) {
        if (by_rows(a.rows, a.vocab, a.top)) {
            const dim3 grid(rows_groups(a.rows)), block(kRowsThreads);
            constexpr int PER_16 = 16 / Vec<T>::N;
            if (a.vocab <= 32) hipLaunchKernelGGL((k_logprobs_rows<T, 2 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
            else if (a.vocab <= 48) hipLaunchKernelGGL((k_logprobs_rows<T, 3 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
            else hipLaunchKernelGGL((k_logprobs_rows<T, 4 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
        } else {
            const int vectors = (a.vocab + Vec<T>::N - 1) / Vec<T>::N;   // 16 lanes up to 32 of them
            in_launches(a, vectors <= 32 ? 16 : 4, [&](const LpArgs& b, dim3 grid) {
                if (vectors <= 16) hipLaunchKernelGGL((k_logprobs_short<T, 16, 1, MASK>), grid, dim3(256), 0, st, b);
                else if (vectors <= 32) hipLaunchKernelGGL((k_logprobs_short<T, 16, 2, MASK>), grid, dim3(256), 0, st, b);
                else if (vectors <= 64) hipLaunchKernelGGL((k_logprobs_short<T, 64, 1, MASK>), grid, dim3(256), 0, st, b);
                else hipLaunchKernelGGL((k_logprobs_short<T, 64, 2, MASK>), grid, dim3(256), 0, st, b);
            });
        }
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
        if (by_rows(a.rows, a.vocab, a.top)) {
            const dim3 grid(rows_groups(a.rows)), block(kRowsThreads);
            constexpr int PER_16 = 16 / Vec<T>::N;
            if (a.vocab <= 32) hipLaunchKernelGGL((k_logprobs_grad_rows<T, 2 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
            else if (a.vocab <= 48) hipLaunchKernelGGL((k_logprobs_grad_rows<T, 3 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
            else hipLaunchKernelGGL((k_logprobs_grad_rows<T, 4 * PER_16, MASK>), grid, block, rows_lds(a.vocab), st, a);
        } else {
            const int vectors = (a.vocab + Vec<T>::N - 1) / Vec<T>::N;   // 16 lanes up to 32 of them
            in_launches(a, vectors <= 32 ? 16 : 4, [&](const LpGradArgs& b, dim3 grid) {
                if (vectors <= 16) hipLaunchKernelGGL((k_logprobs_grad_short<T, 16, 1, MASK>), grid, dim3(256), 0, st, b);
                else if (vectors <= 32) hipLaunchKernelGGL((k_logprobs_grad_short<T, 16, 2, MASK>), grid, dim3(256), 0, st, b);
                else if (vectors <= 64) hipLaunchKernelGGL((k_logprobs_grad_short<T, 64, 1, MASK>), grid, dim3(256), 0, st, b);
                else hipLaunchKernelGGL((k_logprobs_grad_short<T, 64, 2, MASK>), grid, dim3(256), 0, st, b);
            });
        }
    } else {
        // a.splits workgroups a row
        const bool in_place = a.x == a.dx;
        const int threads = in_place ? kInPlaceThreads : 256;
        const int64_t most = kMaxGroups / (threads / 256) / a.splits;
        LpGradArgs b = a;
        for (int64_t row0 = 0; row0 < a.rows; row0 += most) {
            b.row0 = (int)row0;
            const dim3 grid((unsigned)((a.rows - row0 < most ? a.rows - row0 : most) * a.splits));
            if (in_place) hipLaunchKernelGGL((k_logprobs_grad<T, MASK, kInPlaceThreads>), grid, dim3(threads), 0, st, b);
            else hipLaunchKernelGGL((k_logprobs_grad<T, MASK, 256>), grid, dim3(threads), 0, st, b);
        }
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
    return part_bytes(rows, plan_forward(rows, vocab, 4, top).splits, top);   // splits do not depend on the type
}

int cfp_token_logprobs(const void* d_logits, int dtype, int64_t ld, int rows, int vocab, const int32_t* d_tokens,
                       const uint8_t* d_mask, int64_t ld_mask, float* d_logprobs, float* d_entropy, int top,
                       int32_t* d_top_ids, float* d_top_logprobs, float* d_stats, void* d_work,
                       size_t work_bytes, void* stream) {
    if (check_rows("cfp_token_logprobs", dtype, d_logits, ld, rows, vocab, d_tokens, d_mask, ld_mask, top)) return 1;
    if (rows == 0) return 0;
    CFP_REQUIRE(d_logprobs, "cfp_token_logprobs: NULL output");
    CFP_REQUIRE(top == 0 || (d_top_ids && d_top_logprobs), "cfp_token_logprobs: top = %d needs both arrays of alternatives", top);
    const LpPlan pl = plan_forward(rows, vocab, (int)elem_bytes(dtype), top);
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
    a.part_top = need ? (uint64_t*)((f4*)d_work + (size_t)rows * pl.splits) : nullptr;
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
    CFP_REQUIRE((d_logits == d_dlogits && (ld == ld_dlogits || rows == 1)) ||
                    apart(d_logits, ld, 0, d_dlogits, ld_dlogits, 0, 1, rows, vocab, elem_bytes(dtype)),
                "cfp_token_logprobs_grad: the gradient may replace the logits, with the same stride, but not overlap them otherwise");
    const LpPlan pl = plan_grad(rows, vocab, (int)elem_bytes(dtype), d_logits == d_dlogits);
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
