// Orthogonalised updates: the nearest semi-orthogonal matrix of a gradient, approached by
// Newton-Schulz products as the Muon optimiser does, alone (cfp_orthogonalize) or with the
// momentum in front and the weight update behind it (cfp_muon_update).  No counterpart in the
// reference, whose only optimiser is Adam (k_adam, craftax_full.cu:10668).
//
//   X_0 = G / (|G|_F + eps), X m x n with m <= n (a tall G is taken transposed), then `steps`
//   times with the step's coefficients (a, b, c):
//     A = X X^T,   B = b A + c A A,   X <- a X + B X
// The polynomial a s + b s^3 + c s^5 acts on every singular value and leaves the singular
// vectors alone.  A and B are symmetric, so of the first two products only the tiles on and
// above the diagonal are computed and each is stored twice: 3 m^2 n + m^3 multiply-adds a step
// counted as two operations, instead of 4 m^2 n + 2 m^3.
//
// Number formats.  Everything between the steps is fp16 on the matrix pipe with fp32
// accumulation, scaled by a power of two so that the range in use sits in the middle of fp16's
// (singular values stay under 1.21 with the standard coefficients; X is held times 2^10, A and
// B times 2^8, so |X| < 64 and |A|, |B| < 256 for other ones):
//   P = 3  every matrix is a pair hi + lo of fp16 numbers (22 bits, X at best to 2^-35) and a
//          product is hi hi + hi lo + lo hi: what is left out, lo lo, is below 2^-22 of a
//          product.  Error against 64 bits about 1e-6 of the result's norm, as fp32 has.
//          What every input type gets unless the caller asks for less.
//   P = 1  one fp16 product; X alone keeps its lo part, for the term a X.  Without it the
//          rounding of X at every step is amplified by a (3.44) a step where singular values
//          are small: 5e-3 of the norm measured instead of 1 to 2e-3.  A third of the matrix
//          instructions (4096 x 4096 bf16: 1.46 ms, 3.53 with three), and only where the caller
//          says so: what it loses, 7e-4 of the norm before the result is rounded, shows beside
//          a bf16 rounding (1.66e-3; together 1.80e-3).
#include <utility>

#include "cfp_internal.h"

namespace cfp {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));

constexpr float kScaleX = 1024.0f, kScaleA = 256.0f;
constexpr int kMaxSteps = 16;
constexpr int kMaxNormGroups = 1024;   // partial sums of squares a matrix

// Matrices are stored in pieces of 16 rows x 32 values, 1 KiB each and contiguous, the pieces of
// 16 rows behind each other: a piece is what one wavefront copies to LDS with one instruction.
// P = 3: the 32 values of a row are the hi parts of 16 entries, then their lo parts (kLo further).
// ld: values a row, a multiple of 64.
constexpr int kPiece = 512, kLo = 16;
template <int P>
__device__ __forceinline__ size_t at(size_t row, int ld, int k) {
    const size_t piece = (row >> 4) * (size_t)(ld >> 5) + (P == 3 ? k >> 4 : k >> 5);
    return piece * kPiece + (row & 15) * 32 + (P == 3 ? k & 15 : k & 31);
}
__device__ __forceinline__ void split_hl(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// What prepares X: the update u whose polar factor is wanted is G, or with a momentum buffer
// m <- beta m + g, u = g + beta m (nesterov) or m.
struct InArgs {
    const void* g;
    int dtype;
    int64_t ld, stride;
    int rows, cols;
    int vec;             // rows start and end on four-element boundaries
    float* mom;          // or null; same ld and stride as g
    float beta;
    int nesterov;
    float* g_clear;      // or null: zeroed behind its last read
    double* part;        // [batch][groups]
    int groups;
    float eps;
};
__device__ __forceinline__ float load_any(const void* p, int dtype, size_t i) {
    return dtype == CFP_F32 ? ((const float*)p)[i]
                            : dtype == CFP_BF16 ? (float)((const __bf16*)p)[i] : (float)((const _Float16*)p)[i];
}
// N pieces of four entries, at i[k] + e * HOP: entry e of piece k exists when e < count[k].  Without
// a branch between the loads, so that all are in flight together: entries that do not exist are read
// from `any` (an entry that does) and replaced by zero.  Vectors (HOP = 1) exist whole or not at all.
template <int N, int HOP>
__device__ __forceinline__ void load_pieces(const void* p, int dtype, bool vec, const size_t (&i)[N], const int (&count)[N],
                                            size_t any, f4 (&v)[N]) {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    if (vec && dtype == CFP_F32) {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = *reinterpret_cast<const f4*>((const float*)p + (count[k] > 0 ? i[k] : any));
    } else if (vec) {
        u2 raw[N];
#pragma unroll
        for (int k = 0; k < N; k++) raw[k] = *reinterpret_cast<const u2*>((const _Float16*)p + (count[k] > 0 ? i[k] : any));
#pragma unroll
        for (int k = 0; k < N; k++)
            v[k] = dtype == CFP_BF16 ? __builtin_convertvector(__builtin_bit_cast(b4, raw[k]), f4)
                                     : __builtin_convertvector(__builtin_bit_cast(h4, raw[k]), f4);
    } else if (dtype == CFP_F32) {
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = ((const float*)p)[e < count[k] ? i[k] + e * HOP : any];
    } else {
        _Float16 raw[N][4];
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) raw[k][e] = ((const _Float16*)p)[e < count[k] ? i[k] + e * HOP : any];
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = dtype == CFP_BF16 ? (float)__builtin_bit_cast(__bf16, raw[k][e]) : (float)raw[k][e];
    }
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[k][e] = e < count[k] ? v[k][e] : 0.0f;
}
__device__ __forceinline__ void store_four(float* p, size_t i, int count, bool vec, const f4& v) {
    if (vec && count >= 4) { *reinterpret_cast<f4*>(p + i) = v; return; }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < count) p[i + e] = v[e];
}

// First pass: momentum and the sum of squares (64 bits: squares of fp32 values neither
// overflow nor vanish).  A wavefront takes 256 columns of a row at a time.
__global__ __launch_bounds__(256) void k_ortho_norm(InArgs a) {
    __shared__ double ws[4];
    const size_t base = (size_t)blockIdx.y * a.stride;
    const unsigned segs = (unsigned)(a.cols + 255) / 256, units = (unsigned)a.rows * segs;
    const int lane = threadIdx.x & 63;
    double s = 0.0;
    // two pieces at a time, all loads before the first use (with the momentum of a 1000 x 2731 fp32
    // matrix, 33 MB: 8 us; one at a time, four neighbouring entries a lane and a branch around each
    // load: 15)
    const unsigned hop = (unsigned)a.groups * 4;
    for (unsigned u0 = blockIdx.x * 4 + (threadIdx.x >> 6); u0 < units; u0 += 2 * hop) {
        f4 v[2], m[2];
        size_t at_g[2];
        int count[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const unsigned u = u0 + k * hop, r = u / segs;
            // rows on four-element boundaries: four entries a lane; others: every 64th
            const int c = (int)(u - r * segs) * 256 + (a.vec ? 4 : 1) * lane;
            count[k] = u < units ? a.vec ? a.cols - c : (a.cols - c + 63) >> 6 : 0;
            at_g[k] = base + (size_t)r * a.ld + c;
        }
        if (a.vec) load_pieces<2, 1>(a.g, a.dtype, true, at_g, count, base, v);
        else load_pieces<2, 64>(a.g, a.dtype, false, at_g, count, base, v);
        if (a.mom) {
            if (a.vec) load_pieces<2, 1>(a.mom, CFP_F32, true, at_g, count, base, m);
            else load_pieces<2, 64>(a.mom, CFP_F32, false, at_g, count, base, m);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if (a.mom) {
                m[k] = a.beta * m[k] + v[k];
                if (a.vec) {
                    store_four(a.mom, at_g[k], count[k], true, m[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e < count[k]) a.mom[at_g[k] + 64 * e] = m[k][e];
                }
                v[k] = a.nesterov ? v[k] + a.beta * m[k] : m[k];
            }
#pragma unroll
            for (int e = 0; e < 4; e++) s += (double)v[k][e] * (double)v[k][e];
        }
    }
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) ws[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[(size_t)blockIdx.y * a.groups + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// The matrices of one call.  All live in the workspace, padded with zeros to whole tiles, which
// the products keep zero; no kernel below needs a bounds check but the last store.
struct Work {
    _Float16* x;        // [batch][mp][ldn]   X
    _Float16* y[2];     // [batch][np][ldm]   X transposed, before and after a step
    _Float16* y_lo;     // [batch][np][ldm]   P = 1: what X transposed lost in its rounding
    _Float16* a;        // [batch][mp][ldm]
    _Float16* b;        // [batch][mp][ldm]
    int mp, np, ldm, ldn;
};

// kScaleX / (|u| + eps) from the sum of squares, in 64 bits: the reciprocal of a norm below 3e-36 is
// past fp32.  0 for a zero matrix without eps.  An infinity among the entries makes it NaN, as NaN
// does: every entry of X then is, not only that one (inf * 0).
__device__ __forceinline__ double scale_of(double squares, float eps) {
    const double norm = sqrt(squares) + (double)eps;
    return norm == 0.0 ? 0.0 : isinf(squares) ? (double)NAN : (double)kScaleX / norm;
}

// Second pass: X = u / (|u| + eps) times kScaleX in both orders, zeros in the padding.  A thread
// takes four consecutive entries of four rows of a 64 x 64 tile, then of its transpose.
template <int P>
__global__ __launch_bounds__(256) void k_ortho_load(InArgs a, Work w, int tall) {
    __shared__ float tile[64][65];
    __shared__ double ws[4];
    const int bt = blockIdx.z;
    const size_t base = (size_t)bt * a.stride;
    // G's rows and columns, padded
    const int r0 = (int)blockIdx.y * 64, c0 = (int)blockIdx.x * 64;
    const int x4 = 4 * (threadIdx.x & 15), y = threadIdx.x >> 4;
    f4 u[4];
    size_t from[4];
    int have[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int r = r0 + 16 * k + y, c = c0 + x4;
        have[k] = r < a.rows ? a.cols - c : 0;
        from[k] = base + (size_t)r * a.ld + c;
    }
    load_pieces<4, 1>(a.g, a.dtype, a.vec, from, have, base, u);
    if (a.mom) {
        f4 m[4];
        load_pieces<4, 1>(a.mom, CFP_F32, a.vec, from, have, base, m);
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = a.nesterov ? u[k] + a.beta * m[k] : m[k];
    }
    double s = 0.0;
    for (int i = threadIdx.x; i < a.groups; i += 256) s += a.part[(size_t)bt * a.groups + i];
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
    __syncthreads();
    const double inv = scale_of((ws[0] + ws[1]) + (ws[2] + ws[3]), a.eps);
    _Float16* d1 = tall ? w.y[0] + (size_t)bt * w.np * w.ldm : w.x + (size_t)bt * w.mp * w.ldn;
    _Float16* d2 = tall ? w.x + (size_t)bt * w.mp * w.ldn : w.y[0] + (size_t)bt * w.np * w.ldm;
    const int ld1 = tall ? w.ldm : w.ldn, ld2 = tall ? w.ldn : w.ldm;
    _Float16* lo = P == 1 ? w.y_lo + (size_t)bt * w.np * w.ldm : nullptr;
    auto put = [&](_Float16* d, int ld, int r, int c, const f4& v, bool keep_lo) __attribute__((always_inline)) {
        h4 hi, lw;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            _Float16 p, q;
            split_hl(v[e], p, q);
            hi[e] = p; lw[e] = q;
        }
        const size_t o = at<P>(r, ld, c);
        *reinterpret_cast<h4*>(d + o) = hi;
        if (P == 3) *reinterpret_cast<h4*>(d + o + kLo) = lw;
        else if (keep_lo) *reinterpret_cast<h4*>(lo + o) = lw;
    };
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int r = r0 + 16 * k + y, c = c0 + x4;
        if (a.g_clear) store_four(a.g_clear, from[k], have[k], a.vec, f4{0.0f, 0.0f, 0.0f, 0.0f});
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = (float)((double)u[k][e] * inv);
            tile[16 * k + y][x4 + e] = v[e];
        }
        put(d1, ld1, r, c, v, tall);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) {
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = tile[x4 + e][16 * k + y];
        put(d2, ld2, c0 + 16 * k + y, r0 + x4, v, !tall);
    }
}

// What becomes of the last step's X: stored as the result, or subtracted from a weight
// (w <- w (1 - lr wd) - lr scale X).
struct OutArgs {
    void* out;
    int dtype;
    int64_t ld, stride;
    int rows, cols, tall;
    int update;          // 0: out = X; 1: out (fp32) is the weight
    const float* lr_dev; // or null
    float lr, decay, scale;
};
__device__ __forceinline__ void put_out(const OutArgs& o, size_t i, float v) {
    if (o.update) {
        const float lr = o.lr_dev ? o.lr * *o.lr_dev : o.lr;
        float* w = (float*)o.out + i;
        *w = *w * (1.0f - lr * o.decay) - lr * o.scale * v;
    } else if (o.dtype == CFP_F32) {
        ((float*)o.out)[i] = v;
    } else if (o.dtype == CFP_BF16) {
        ((__bf16*)o.out)[i] = (__bf16)v;
    } else {
        ((_Float16*)o.out)[i] = (_Float16)v;
    }
}

// rows row0, row0 + 2, ... + 14, one column a lane
__device__ __forceinline__ void put_rows(const OutArgs& o, size_t base, int row0, int col, const float (&v)[8]) {
    if (col >= o.cols) return;
    const size_t i = base + (size_t)row0 * o.ld + col, hop = 2 * (size_t)o.ld;
    if (o.update) {
        const float lr = o.lr_dev ? o.lr * *o.lr_dev : o.lr, keep = 1.0f - lr * o.decay, step = lr * o.scale;
        float* w = (float*)o.out;
        float old[8];
#pragma unroll
        for (int k = 0; k < 8; k++) old[k] = row0 + 2 * k < o.rows ? w[i + k * hop] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (row0 + 2 * k < o.rows) w[i + k * hop] = old[k] * keep - step * v[k];
    } else if (o.dtype == CFP_F32) {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (row0 + 2 * k < o.rows) ((float*)o.out)[i + k * hop] = v[k];
    } else if (o.dtype == CFP_BF16) {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (row0 + 2 * k < o.rows) ((__bf16*)o.out)[i + k * hop] = (__bf16)v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (row0 + 2 * k < o.rows) ((_Float16*)o.out)[i + k * hop] = (_Float16)v[k];
    }
}

// ---- the product C[i][j] = sum_k L[i][k] R[j][k] and what is made of it ---------------
enum { kGram, kPoly, kStep, kLast };
constexpr int kBlockWaves = 8;   // of k_ortho_block
struct MulArgs {
    const _Float16* l;
    const _Float16* r;
    int ldl, ldr;            // values (hi and lo counted apart) a row
    size_t l_batch, r_batch; // values a matrix
    int stages;              // of 32 values; even
    int tiles_i;
    int tiles;               // of one matrix
    int runs;                // an XCD takes a run of tiles
    unsigned row_len;        // tiles of a pair of rows (symmetric products), of a column, or of a band
    uint64_t row_inv;        // ceil(2^32 / row_len)
    int by_xcd;              // 0, or the matrices of the batch where one XCD takes each
    Work w;
    int cur;                 // y[cur] is X transposed before the step
    float a, b, c;
    OutArgs out;
    // X X^T of few tiles and many stages: the stages shared out over `splits` workgroups a tile
    int splits;
    f4* part;                // [batch][tile][split][4 wavefronts][4][64 lanes]
};
__device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Loads the arguments that lead to a workgroup's first copies at once: left to the branches that
// use them they are five loads one after the other (0.25 us a launch).
__device__ __forceinline__ void load_args(const MulArgs& g) {
    asm volatile("" ::"s"(g.l), "s"(g.r), "s"(g.ldl), "s"(g.ldr), "s"(g.l_batch), "s"(g.r_batch), "s"(g.stages), "s"(g.tiles_i),
                 "s"(g.tiles), "s"(g.runs), "s"(g.row_len), "s"(g.row_inv), "s"(g.by_xcd), "s"(g.splits));
}

// Waits until at most min(later, MOST) * LOADS of this wave's copies are in flight.  Copies are
// the only vector-memory operations between the prologue and the epilogue, so the counts are
// those of the source.
template <int LOADS, int MOST>
__device__ __forceinline__ void wait_copies(int later) {
    if (MOST >= 1 && later >= MOST) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS * MOST) : "memory");
    } else if constexpr (MOST > 1) {
        wait_copies<LOADS, MOST - 1>(later);
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
}

// Dwords 0, 1 of this lane and 2, 3 of lane - 32 (the lower half keeps 0, 1 and gets 0, 1 of lane
// + 32 as its 2, 3): what turns 16 contiguous bytes of a row into the 8-byte pieces of two q, and
// back.
__device__ __forceinline__ void swap_halves(u4& v) {
#pragma unroll
    for (int d = 0; d < 2; d++) {
        const auto r = __builtin_amdgcn_permlane32_swap(v[d], v[2 + d], false, false);
        v[d] = r[0];
        v[2 + d] = r[1];
    }
}
__device__ __forceinline__ float half_of(const u4& v, int i) {
    return (float)__builtin_bit_cast(h8, v)[i];
}
// Lane c of a quad holds entries (0..3, c) of a 4 x 4 matrix of fp16, two a dword; afterwards
// entries (c, 0..3).
__device__ __forceinline__ u2 transpose_quad(u2 w, int c) {
    const unsigned sel = c & 1 ? 0x03020706u : 0x05040100u;   // odd: (other hi, own hi), even: (own lo, other lo)
    u2 r;
#pragma unroll
    for (int d = 0; d < 2; d++) {
        const unsigned other = __builtin_amdgcn_mov_dpp(w[d], 0xb1, 0xf, 0xf, true);   // lane ^ 1
        r[d] = __builtin_amdgcn_perm(other, w[d], sel);
    }
    const bool low = (c & 2) == 0;
    const unsigned got = __builtin_amdgcn_mov_dpp(low ? r[1] : r[0], 0x4e, 0xf, 0xf, true);   // lane ^ 2
    return low ? u2{r[0], got} : u2{got, r[1]};
}

// ---- what becomes of a 32 x 32 block of the product -------------------------------------
// A lane holds column n32 of the block, rows 8 q + 4 half + 0..3 (q = 0..3).  Transposed
// matrices (rows j) are read and written 16 bytes a lane: lanes n32 and n32 + 32 hold
// neighbouring 8-byte pieces, of q = 2 t and 2 t + 1, and swap two of the four dwords.
// What is added to the product: X transposed (with its lo part), or A.
struct Addend {
    u4 v[2][2];   // [t][hi, lo]
};
template <int P, int MODE>
__device__ __forceinline__ void load_addend(const MulArgs& g, size_t bt, int ib, int jb, int lane, Addend& a) {
    if (MODE == kGram) return;
    const int j = jb + (lane & 31), half = lane >> 5;
    const size_t mat_y = bt * g.w.np * (size_t)g.w.ldm;
    const _Float16* m = MODE == kPoly ? g.w.a + bt * g.w.mp * (size_t)g.w.ldm : g.w.y[g.cur] + mat_y;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const size_t o = at<P>(j, g.w.ldm, ib + 16 * t) + 8 * half;
        a.v[t][0] = *reinterpret_cast<const u4*>(m + o);
        if (P == 3) a.v[t][1] = *reinterpret_cast<const u4*>(m + o + kLo);
        else if (MODE != kPoly) a.v[t][1] = *reinterpret_cast<const u4*>(g.w.y_lo + mat_y + o);
    }
}
template <int P, int MODE>
__device__ __forceinline__ void finish_block(const MulArgs& g, size_t bt, const f16v& acc, Addend& add, int ib, int jb, int lane,
                                             bool diagonal, float (*out_stage)[33]) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly, HAS_LO = P == 3 || !SYM;
    const int n32 = lane & 31, half = lane >> 5, quad = lane & 3, j = jb + n32;
    const size_t mat_a = bt * g.w.mp * (size_t)g.w.ldm, mat_y = bt * g.w.np * (size_t)g.w.ldm;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        if (MODE != kGram) {
            swap_halves(add.v[t][0]);
            if (HAS_LO) swap_halves(add.v[t][1]);
        }
        u4 hi_out, lo_out;   // dwords 0, 1: q = 2 t; 2, 3: q = 2 t + 1
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int q = 2 * t + u;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = acc[4 * q + e];
                float x = 0.0f;
                if (MODE != kGram) {
                    x = half_of(add.v[t][0], 4 * u + e);
                    if (HAS_LO) x += half_of(add.v[t][1], 4 * u + e);
                }
                if (MODE == kGram) v[e] *= kScaleA / (kScaleX * kScaleX);
                else if (MODE == kPoly) v[e] = g.b * x + (g.c / kScaleA) * v[e];
                else v[e] = g.a * x + v[e] * (1.0f / kScaleA);
            }
            if (MODE == kLast) {
#pragma unroll
                for (int e = 0; e < 4; e++) out_stage[8 * q + 4 * half + e][n32] = v[e] * (1.0f / kScaleX);
                continue;
            }
            h4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                _Float16 p, r;
                split_hl(v[e], p, r);
                hi[e] = p; lo[e] = r;
            }
            const u2 hw = __builtin_bit_cast(u2, hi), lw = __builtin_bit_cast(u2, lo);
            hi_out[2 * u] = hw[0]; hi_out[2 * u + 1] = hw[1];
            lo_out[2 * u] = lw[0]; lo_out[2 * u + 1] = lw[1];
            // row-major: four lanes exchange their columns, one row of four entries each
            _Float16* to = MODE == kGram ? g.w.a + mat_a : MODE == kPoly ? g.w.b + mat_a
                                                                         : g.w.x + bt * g.w.mp * (size_t)g.w.ldn;
            to += at<P>(ib + 8 * q + 4 * half + quad, SYM ? g.w.ldm : g.w.ldn, jb + (n32 & 28));
            *reinterpret_cast<u2*>(to) = transpose_quad(hw, quad);
            if (P == 3) *reinterpret_cast<u2*>(to + kLo) = transpose_quad(lw, quad);
        }
        if (MODE == kLast) continue;
        // a tile on the diagonal holds both halves itself, and has stored them
        if (SYM && diagonal) continue;
        const size_t o = at<P>(j, g.w.ldm, ib + 16 * t) + 8 * half;
        _Float16* to = SYM ? (MODE == kGram ? g.w.a : g.w.b) + mat_a : g.w.y[g.cur ^ 1] + mat_y;
        swap_halves(hi_out);
        *reinterpret_cast<u4*>(to + o) = hi_out;
        if (HAS_LO) {
            swap_halves(lo_out);
            *reinterpret_cast<u4*>(P == 3 ? to + o + kLo : g.w.y_lo + mat_y + o) = lo_out;
        }
    }
}
// rows of 32 values of the result, two a wavefront and instruction, eight in flight
__device__ __forceinline__ void write_result(const OutArgs& o, size_t bt, int ib, int jb, int lane, const float (*out_stage)[33]) {
#pragma unroll 1
    for (int b = 0; b < 2; b++) {
        const int n32 = lane & 31, p0 = 16 * b + (lane >> 5);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = o.tall ? out_stage[n32][p0 + 2 * k] : out_stage[p0 + 2 * k][n32];
        put_rows(o, bt * o.stride, (o.tall ? jb : ib) + p0, (o.tall ? ib : jb) + n32, v);
    }
}

// f(0), f(1), ... with compile-time numbers (a loop of 48 steps is not unrolled whole)
template <class Fn, int... I>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, Fn&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}

// Tile of number t.  In scalar arithmetic throughout (addresses of copies are scalar operands):
// t / d as t * ceil(2^32 / d) / 2^32, exact while t * d < 2^32.
template <bool SYM>
__device__ __forceinline__ void tile_of(const MulArgs& g, unsigned t, int& ti, int& tj) {
    if (g.runs) {
        const unsigned x = t % 8, q = (unsigned)g.tiles / 8, r = (unsigned)g.tiles % 8;
        t = x * q + (x < r ? x : r) + t / 8;
    }
    if (SYM) {
        // tiles on and above the diagonal: row r and row n - 1 - r have n + 1 of them together
        const unsigned row = (unsigned)((t * g.row_inv) >> 32), col = t - row * g.row_len;
        const int n = g.tiles_i, r = (int)row, c = (int)col;
        ti = c < n - r ? r : n - 1 - r;
        tj = c < n - r ? r + c : c - 1;
    } else if (!g.runs) {   // column by column
        const unsigned col = (unsigned)((t * g.row_inv) >> 32);
        ti = (int)(t - col * g.row_len);
        tj = (int)col;
    } else {                // bands of four tile rows, each column by column
        const unsigned band = (unsigned)((t * g.row_inv) >> 32), rest = t - band * g.row_len;
        const unsigned rows = (unsigned)g.tiles_i - 4 * band;   // of the last band: 1 to 4
        const unsigned col = rows >= 4 ? rest >> 2 : rows == 3 ? (rest * 43691u) >> 17 : rows == 2 ? rest >> 1 : rest;
        ti = (int)(4 * band + rest - col * (rows >= 4 ? 4 : rows));
        tj = (int)col;
    }
}

// 2 x 2 wavefronts of F x F blocks of 32 x 32 (tiles of 64 F).  A stage is SUB times 32 values of
// every row of the tile's L and R sides, copied to LDS without registers (each lane's 16 bytes
// land at the wave's base + 16 * lane) into a ring of R buffers.  16-byte chunk c of row r sits at
// chunk c ^ (r / 4 & 3): the chunks of sixteen consecutive rows then cover all 64 banks.
// A group is the matrix instructions of 16 of the K entries (P = 1: 32 values are two groups, P = 3:
// one of three times as many); its operands are read from LDS while the group before it
// multiplies, in an order that is pinned: left to itself the compiler reuses the operand registers
// at once and waits for every read (615 instead of 1000 TFLOP/s at 4096 x 4096).
template <int P, int MODE, int F, int SUB, int R>
__global__ __launch_bounds__(256) void k_ortho_mul(MulArgs g) {
    constexpr int T = 64 * F, WAVES = 4;
    constexpr int LOADS = SUB * 2 * T / 16 / WAVES;   // pieces a wave and stage
    constexpr int GROUPS = SUB * (P == 3 ? 1 : 2);
    static_assert(GROUPS % 2 == 0 && LOADS % GROUPS == 0, "operand sets alternate; copies are spread evenly");
    constexpr int PL = P == 3 ? 2 : 1;
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    constexpr int NM = (P == 3 ? 3 : 1) * F * F, NR = 2 * PL * F;
    __shared__ __align__(1024) unsigned char lds[R][SUB][2 * T * 64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n32 = lane & 31, half = lane >> 5;
    load_args(g);
    // by_xcd: blockIdx.y and the residue of blockIdx.x (the XCD) name the matrix
    const unsigned tile = g.by_xcd ? blockIdx.x / 8 : blockIdx.x;
    const size_t bt = g.by_xcd ? blockIdx.y * 8 + blockIdx.x % 8 : blockIdx.y;
    if (g.by_xcd && (int)bt >= g.by_xcd) return;
    int ti, tj;
    tile_of<SYM>(g, tile, ti, tj);
    const int i0 = ti * T, j0 = tj * T;
    // this wave's pieces of stage 0: F of the L side, F of the R side
    const _Float16* from[2] = {g.l + bt * g.l_batch + (size_t)(i0 / 16 + wave) * (g.ldl >> 5) * kPiece,
                               g.r + bt * g.r_batch + (size_t)(j0 / 16 + wave) * (g.ldr >> 5) * kPiece};
    const size_t hop[2] = {(size_t)WAVES * (g.ldl >> 5) * kPiece, (size_t)WAVES * (g.ldr >> 5) * kPiece};
    const unsigned voff = (unsigned)((lane >> 2) * 64 + ((lane & 3) ^ ((lane >> 4) & 3)) * 16);
    constexpr bool SPLIT = MODE == kGram && F == 1;
    int first = 0, last = g.stages / SUB - 1;   // stages of this workgroup
    if (SPLIT) {
        const unsigned all = (unsigned)(last + 1), z = blockIdx.z;
        first = (int)(all * z / (unsigned)g.splits);
        last = (int)(all * (z + 1) / (unsigned)g.splits) - 1 - first;
    }
    // copy q of a stage into ring buffer `buf`: sub-stage by sub-stage, the L side first
    auto copy = [&](int stage, int buf, int q) __attribute__((always_inline)) {
        constexpr int HALF = LOADS / SUB / 2;
        const int sub = q / (2 * HALF), side = q / HALF % 2, i = q % HALF;
        const unsigned to = (unsigned)(size_t)&lds[buf][sub][(side * T + (i * WAVES + wave) * 16) * 64];
        asm volatile(
            "s_mov_b32 m0, %2\n\t"
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, %1"
            :
            : "v"(voff + (unsigned)((first + stage) * SUB + sub) * (kPiece * 2)), "s"(from[side] + i * hop[side]), "s"(to)
            : "memory", "m0");
    };

    // F = 1 has one block a wavefront: products of different planes or K steps go to accumulators
    // of their own, or each matrix instruction would wait for the one before it.
    constexpr int ACCS = F > 1 ? 1 : P == 3 ? 3 : 2;
    f16v acc[F][F][ACCS];
#pragma unroll
    for (int i = 0; i < F * F * ACCS; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i / (F * ACCS)][i / ACCS % F][i % ACCS][e] = 0.0f;
    const int wi = (wave & 1) * F * 32, wj = (wave >> 1) * F * 32;
    // operand registers of two groups: [group][plane][side][block]
    h8 op[2][PL][2][F];
    const int chunk_of[2] = {(half ^ ((n32 >> 2) & 3)) * 16, ((2 + half) ^ ((n32 >> 2) & 3)) * 16};
    // operand t of group `gr` of the stage in buffer `buf`, in the order of use: the hi planes
    // first, L and R in turn
    auto read = [&](int buf, int gr, int t) __attribute__((always_inline)) {
        const int sub = P == 3 ? gr : gr / 2, z = t / (2 * F), side = t % 2, b = (t % (2 * F)) / 2;
        const int row = side * T + (side ? wj : wi) + 32 * b + n32;
        op[gr % 2][z][side][b] = *reinterpret_cast<const h8*>(&lds[buf][sub][row * 64 + chunk_of[P == 3 ? z : gr % 2]]);
    };
    auto multiply = [&](int gr, int m) __attribute__((always_inline)) {
        const int z = m / (F * F), i = (m % (F * F)) / F, j = m % F;   // z: hi hi, hi lo, lo hi
        f16v& to = acc[i][j][ACCS == 1 ? 0 : P == 3 ? z : gr % 2];
        to = mma(op[gr % 2][z == 2 ? PL - 1 : 0][0][i], op[gr % 2][z == 1 ? PL - 1 : 0][1][j], to);
    };
    // Group `gr`: its matrix instructions, one LDS read of the next group's operands (next_buf)
    // behind each of the first ones, and its share of the copies of stage `stage` into buffer
    // `free_buf` spread over it (a burst of copies fills the address unit's queue and stops the
    // wave).
    auto group = [&](auto at_gr, auto reading, auto copying, int next_buf, int stage, int free_buf, int share)
                     __attribute__((always_inline)) {
        constexpr int gr = decltype(at_gr)::value, next = (gr + 1) % GROUPS, Q = LOADS / GROUPS;
        __builtin_amdgcn_sched_barrier(0);
        each(std::make_integer_sequence<int, NM>{}, [&](auto at_m) __attribute__((always_inline)) {
            constexpr int m = decltype(at_m)::value;
            multiply(gr, m);
            if (decltype(reading)::value)
#pragma unroll
                for (int t = m * NR / NM; t < (m + 1) * NR / NM; t++) read(next_buf, next, t);
            if (decltype(copying)::value)
#pragma unroll
                for (int q = m * Q / NM; q < (m + 1) * Q / NM; q++) copy(stage, free_buf, share * Q + q);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    using std::integral_constant;
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    // Stage s from its last group on to the last but one of stage s + 1.  Before that group reads
    // stage s + 1: this wave's copies of it have landed, behind the barrier everyone's have; and
    // everyone has read all of stage s, whose buffer takes stage s + R.
    auto advance = [&](auto copying, int s, int buf, int nb, int later) __attribute__((always_inline)) {
        wait_copies<LOADS, R - 2>(later);
        __syncthreads();
        group(integral_constant<int, GROUPS - 1>{}, yes, copying, nb, s + R, buf, 0);
        each(std::make_integer_sequence<int, GROUPS - 1>{}, [&](auto at) __attribute__((always_inline)) {
            group(at, yes, copying, nb, s + R, buf, decltype(at)::value + 1);
        });
    };
    for (int s = 0; s < R && s <= last; s++)
#pragma unroll
        for (int q = 0; q < LOADS; q++) copy(s, s, q);
    wait_copies<LOADS, R - 1>(last);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NR; t++) read(0, 0, t);
    each(std::make_integer_sequence<int, GROUPS - 1>{}, [&](auto at) __attribute__((always_inline)) {
        group(at, yes, no, 0, 0, 0, 0);
    });
    int buf = 0, s = 0;
    for (; s + R <= last; s++) {
        const int nb = buf == R - 1 ? 0 : buf + 1;
        advance(yes, s, buf, nb, R - 2);
        buf = nb;
    }
    for (; s < last; s++) {
        const int nb = buf == R - 1 ? 0 : buf + 1;
        advance(no, s, buf, nb, last - s - 1);
        buf = nb;
    }
    group(integral_constant<int, GROUPS - 1>{}, no, no, 0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < F * F; i++)
#pragma unroll
        for (int z = 1; z < ACCS; z++) acc[i / F][i % F][0] += acc[i / F][i % F][z];

    if (SPLIT && g.splits > 1) {   // k_ortho_fold adds the parts up
        f4* part = g.part + (((bt * g.tiles + tile) * g.splits + blockIdx.z) * 4 + wave) * 256 + lane;
#pragma unroll
        for (int e = 0; e < 4; e++)
            part[64 * e] = f4{acc[0][0][0][4 * e], acc[0][0][0][4 * e + 1], acc[0][0][0][4 * e + 2], acc[0][0][0][4 * e + 3]};
        return;
    }

    // ---- epilogue
    // The last step's values leave through LDS, a block column of the wavefront at a time: whole
    // rows of the result in either order.  Its operands are read (barrier).
    float (*out_stage)[32][33] = reinterpret_cast<float (*)[32][33]>(&lds[0][0][0] + wave * (F * 32 * 33 * 4));
    static_assert(sizeof(lds) >= 4 * F * 32 * 33 * 4, "the stage of the results fits into the ring");
    if (MODE == kLast) __syncthreads();
    const int end_i = g.w.mp, end_j = SYM ? g.w.mp : g.w.np;
    constexpr int BATCH = F == 4 ? 1 : F;   // blocks whose addends are loaded together; more do not
                                            // fit beside 256 accumulators
#pragma unroll
    for (int fj = 0; fj < F; fj++) {
        const int jb = j0 + wj + 32 * fj;
        if (jb >= end_j) continue;   // whole blocks: the ends are multiples of 64
        Addend add[F];
#pragma unroll
        for (int f0 = 0; f0 < F; f0 += BATCH) {
#pragma unroll
            for (int fi = f0; fi < f0 + BATCH; fi++)
                if (i0 + wi + 32 * fi < end_i) load_addend<P, MODE>(g, bt, i0 + wi + 32 * fi, jb, lane, add[fi]);
#pragma unroll
            for (int fi = f0; fi < f0 + BATCH; fi++)
                if (i0 + wi + 32 * fi < end_i)
                    finish_block<P, MODE>(g, bt, acc[fi][fj][0], add[fi], i0 + wi + 32 * fi, jb, lane, SYM && ti == tj,
                                          out_stage[MODE == kLast ? fi : 0]);
        }
        if (MODE == kLast) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int fi = 0; fi < F; fi++)
                if (i0 + wi + 32 * fi < end_i) write_result(g.out, bt, i0 + wi + 32 * fi, jb, lane, out_stage[fi]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---- the same products where they leave most CUs idle ----------------------------------------
// A workgroup makes one 32 x 32 block and its wavefronts share out the K axis: every wavefront
// reads operands of its own, from L2 straight into registers, the parts meet in LDS and are added
// in the order of the wavefronts.  Bound by the round trips to memory, one for every four stages of
// a wavefront, and by the launch.  All steps, fp32, with k_ortho_mul / this kernel: 256 x 843
// 104 / 97 us, 500 x 1000 130 / 119, 16 x 128 x 512 78 / 73.
template <int P, int MODE>
__global__ __launch_bounds__(64 * kBlockWaves) void k_ortho_block(MulArgs g) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    __shared__ f4 part[kBlockWaves][4][64];
    __shared__ float out_stage[MODE == kLast ? 32 : 1][33];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n32 = lane & 31, half = lane >> 5;
    load_args(g);
    const unsigned tile = g.by_xcd ? blockIdx.x / 8 : blockIdx.x;   // as in k_ortho_mul
    const size_t bt = g.by_xcd ? blockIdx.y * 8 + blockIdx.x % 8 : blockIdx.y;
    if (g.by_xcd && (int)bt >= g.by_xcd) return;
    int ti, tj;
    tile_of<SYM>(g, tile, ti, tj);
    const int first = g.stages * wave / kBlockWaves, count = g.stages * (wave + 1) / kBlockWaves - first;
    // piece of rows n32 / 16, row n32 % 16 of it, entries 8 half and up: a lane's first 16 bytes
    const _Float16* l = g.l + bt * g.l_batch + ((size_t)(2 * ti + (n32 >> 4)) * (g.ldl >> 5) + first) * kPiece + (n32 & 15) * 32 + 8 * half;
    const _Float16* r = g.r + bt * g.r_batch + ((size_t)(2 * tj + (n32 >> 4)) * (g.ldr >> 5) + first) * kPiece + (n32 & 15) * 32 + 8 * half;
    f16v acc[3];
#pragma unroll
    for (int z = 0; z < 3; z++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[z][e] = 0.0f;
    Addend add;
    if (wave == 0) load_addend<P, MODE>(g, bt, ti * 32, tj * 32, lane, add);
    constexpr int U = 4;   // stages whose operands are loaded together
    auto stages = [&](auto many) __attribute__((always_inline)) {
        constexpr int N = decltype(many)::value;
        h8 l0[N], l1[N], r0[N], r1[N];
#pragma unroll
        for (int u = 0; u < N; u++) {
            l0[u] = *reinterpret_cast<const h8*>(l + u * kPiece); l1[u] = *reinterpret_cast<const h8*>(l + u * kPiece + 16);
            r0[u] = *reinterpret_cast<const h8*>(r + u * kPiece); r1[u] = *reinterpret_cast<const h8*>(r + u * kPiece + 16);
        }
#pragma unroll
        for (int u = 0; u < N; u++) {
            acc[0] = mma(l0[u], r0[u], acc[0]);
            if (P == 3) {
                acc[1] = mma(l0[u], r1[u], acc[1]);
                acc[2] = mma(l1[u], r0[u], acc[2]);
            } else {
                acc[1] = mma(l1[u], r1[u], acc[1]);
            }
        }
        l += N * kPiece; r += N * kPiece;
    };
    int s = 0;
    for (; s + U <= count; s += U) stages(std::integral_constant<int, U>{});
    if (count - s >= 2) { stages(std::integral_constant<int, 2>{}); s += 2; }
    if (count - s >= 1) stages(std::integral_constant<int, 1>{});
    acc[0] += acc[1];
    if (P == 3) acc[0] += acc[2];
    if (wave > 0)
#pragma unroll
        for (int e = 0; e < 4; e++) part[wave][e][lane] = f4{acc[0][4 * e], acc[0][4 * e + 1], acc[0][4 * e + 2], acc[0][4 * e + 3]};
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kBlockWaves; w++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const f4 v = part[w][e][lane];
#pragma unroll
            for (int k = 0; k < 4; k++) acc[0][4 * e + k] += v[k];
        }
    finish_block<P, MODE>(g, bt, acc[0], add, ti * 32, tj * 32, lane, ti == tj, out_stage);
    if (MODE == kLast) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        write_result(g.out, bt, ti * 32, tj * 32, lane, out_stage);
    }
}

// The parts of a tile of X X^T, added up in the order of the splits.  (A launch of its own: the
// fences of a last-one-adds scheme inside the product cost 65 to 86 us a launch here, each writes
// back an L2.)
template <int P>
__global__ __launch_bounds__(256) void k_ortho_fold(MulArgs g) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int ti, tj;
    tile_of<true>(g, blockIdx.x, ti, tj);
    const size_t bt = blockIdx.y;
    const f4* p = g.part + ((bt * g.tiles + blockIdx.x) * g.splits * 4 + wave) * 256 + lane;
    f16v sum;
#pragma unroll
    for (int e = 0; e < 16; e++) sum[e] = 0.0f;
#pragma unroll 4
    for (int z = 0; z < g.splits; z++, p += 1024) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const f4 v = p[64 * e];
#pragma unroll
            for (int k = 0; k < 4; k++) sum[4 * e + k] += v[k];
        }
    }
    Addend none;
    finish_block<P, kGram>(g, bt, sum, none, ti * 64 + (wave & 1) * 32, tj * 64 + (wave >> 1) * 32, lane, ti == tj, nullptr);
}

// ---- A A and B X in one launch, for m up to 256 --------------------------------------------
// There a step's three launches are 5 to 7 us each of which the matrix instructions are one: the
// time is that of launches and first loads.  A workgroup makes the 32 rows of B that it needs
// itself (m <= 256: at most as much work as its part of B X) and multiplies them with 128 columns
// of X; B stays in LDS.  Stages of 64 values of A's rows, then of X transposed, go through one
// ring without a break between the products.  MB = m / 64, so every count is known.
// copies that may be in flight when stage s must have landed: those of the stages issued after it
template <int S, int R, int LOADS_A, int LOADS_X>
constexpr int flying(int s) {
    int n = 0;
    for (int t = s + 1; t < s + R - 1 && t < 2 * S; t++) n += t < S ? LOADS_A : LOADS_X;
    return n;
}
template <int P, int MODE, int MB>
__global__ __launch_bounds__(256) void k_ortho_pair(MulArgs g) {
    constexpr int PL = P == 3 ? 2 : 1, S = MB * PL;       // stages of one product, 64 values each
    constexpr int NB = (MB + 1) / 2;                      // blocks of B a wavefront makes at most
    constexpr int LOADS_A = 2 * MB, LOADS_X = 4;          // copies a wavefront and stage
    constexpr int ROWS = MB * 64 > 128 ? MB * 64 : 128;   // of a ring buffer
    constexpr int R = MB > 3 ? 3 : 4;
    constexpr int ACCS = P == 3 ? 3 : 2;
    // own rows of A, then of B in their place: [32 values][32 rows][64 bytes], chunks swizzled as in
    // the ring
    __shared__ __align__(1024) unsigned char own[2 * S][32 * 64], ring[R][2][ROWS * 64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n32 = lane & 31, half = lane >> 5;
    asm volatile("" ::"s"(g.w.a), "s"(g.w.y[0]), "s"(g.w.y[1]), "s"(g.cur), "s"(g.w.mp), "s"(g.w.np), "s"(g.w.ldm), "s"(g.by_xcd));
    const unsigned tile_i = g.by_xcd ? blockIdx.x / 8 : blockIdx.x;   // as in k_ortho_mul
    const size_t bt = g.by_xcd ? blockIdx.z * 8 + blockIdx.x % 8 : blockIdx.z;
    if (g.by_xcd && (int)bt >= g.by_xcd) return;
    const int i0 = (int)tile_i * 32, j0 = (int)blockIdx.y * 128;
    const size_t mat_a = bt * g.w.mp * (size_t)g.w.ldm, mat_y = bt * g.w.np * (size_t)g.w.ldm;
    const unsigned voff = (unsigned)((lane >> 2) * 64 + ((lane & 3) ^ ((lane >> 4) & 3)) * 16);
    auto copy = [&](const _Float16* from, int stage, void* to) __attribute__((always_inline)) {
        asm volatile(
            "s_mov_b32 m0, %2\n\t"
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %0, %1"
            :
            : "v"(voff + (unsigned)stage * (kPiece * 2)), "s"(from), "s"((unsigned)(size_t)to)
            : "memory", "m0");
    };
    const size_t row_of_pieces = (size_t)(2 * S) * kPiece;   // 16 rows of a matrix with ldm = 64 S
    const _Float16* src_a = g.w.a + mat_a + wave * row_of_pieces;
    const _Float16* src_x = g.w.y[g.cur] + mat_y + ((size_t)(j0 / 16) + wave) * row_of_pieces;
    const _Float16* src_own = g.w.a + mat_a + (size_t)(i0 / 16) * row_of_pieces;
    // stages 0 .. S - 1: A; S .. 2 S - 1: X transposed
    auto copy_stage = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            unsigned char* to = ring[s % R][sub];
            if (s < S) {
#pragma unroll
                for (int q = 0; q < MB; q++) copy(src_a + q * 4 * row_of_pieces, 2 * s + sub, to + (q * 4 + wave) * 1024);
            } else {
#pragma unroll
                for (int q = 0; q < 2; q++) copy(src_x + q * 4 * row_of_pieces, 2 * (s - S) + sub, to + (q * 4 + wave) * 1024);
            }
        }
    };
    const int sw = (n32 >> 2) & 3;
    auto operand = [&](const unsigned char* rows, int row0, int chunk) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(rows + (row0 + n32) * 64 + ((chunk + half) ^ sw) * 16);
    };
    // one stage of L (32 own rows) times R (32 rows of the ring buffer) into acc
    auto multiply = [&](const unsigned char* l, const unsigned char* r, int row0, f16v (&acc)[ACCS]) __attribute__((always_inline)) {
        const h8 l0 = operand(l, 0, 0), l1 = operand(l, 0, 2), r0 = operand(r, row0, 0), r1 = operand(r, row0, 2);
        acc[0] = mma(l0, r0, acc[0]);
        if (P == 3) {   // hi and lo of 16 entries
            acc[1] = mma(l0, r1, acc[1]);
            acc[2] = mma(l1, r0, acc[2]);
        } else {        // 32 entries
            acc[1] = mma(l1, r1, acc[1]);
        }
    };
    f16v acc[NB][ACCS];
    auto clear = [](f16v (&a)[ACCS]) __attribute__((always_inline)) {
#pragma unroll
        for (int z = 0; z < ACCS; z++)
#pragma unroll
            for (int e = 0; e < 16; e++) a[z][e] = 0.0f;
    };
    auto total = [](const f16v (&a)[ACCS]) __attribute__((always_inline)) {
        f16v s = a[0];
#pragma unroll
        for (int z = 1; z < ACCS; z++) s += a[z];
        return s;
    };
    // own rows of A first (oldest, so landed whenever a stage of the ring has)
#pragma unroll
    for (int q = 0; q < 4 * S; q += 4) {
        const int piece = q + wave;   // of values 32 (piece / 2) .., rows 16 (piece % 2) ..
        copy(src_own + (piece & 1) * row_of_pieces, piece >> 1, &own[piece >> 1][(piece & 1) * 1024]);
    }
#pragma unroll
    for (int s = 0; s < R - 1; s++)
        if (s < 2 * S) copy_stage(s);
#pragma unroll
    for (int b = 0; b < NB; b++) clear(acc[b]);
    // Stage s has landed for this wavefront and, behind the barrier, for all; and all are done
    // with stage s - 1, whose buffer takes stage s + R - 1.
    auto turn = [&](auto at_s) __attribute__((always_inline)) {
        constexpr int s = decltype(at_s)::value;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(flying<S, R, LOADS_A, LOADS_X>(s)) : "memory");
        __syncthreads();
        if (s + R - 1 < 2 * S) copy_stage(s + R - 1);
    };
    each(std::make_integer_sequence<int, S>{}, [&](auto at_s) __attribute__((always_inline)) {
        constexpr int s = decltype(at_s)::value;
        turn(at_s);
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (wave + 4 * b < 2 * MB) multiply(own[2 * s + sub], ring[s % R][sub], (wave + 4 * b) * 32, acc[b]);
    });
    // B = b A + c A A, own rows, in the form of an operand and in place of A: a wavefront replaces
    // the columns that it alone still reads
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; b++) {
        if (wave + 4 * b >= 2 * MB) continue;
        const int jb = (wave + 4 * b) * 32, quad = lane & 3;
        const f16v sum = total(acc[b]);
        // entry (row, k) of an operand: byte offset of its hi part
        auto place = [&](int row, int k) {
            const int chunk = P == 3 ? (k & 15) >> 3 : (k & 31) >> 3;
            return (P == 3 ? k >> 4 : k >> 5) * (32 * 64) + row * 64 + ((chunk ^ ((row >> 2) & 3)) * 16) + (k & 7) * 2;
        };
        auto place_lo = [&](int row, int k) {
            return (k >> 4) * (32 * 64) + row * 64 + (((2 + ((k & 15) >> 3)) ^ ((row >> 2) & 3)) * 16) + (k & 7) * 2;
        };
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int row = 8 * (e >> 2) + 4 * half + (e & 3);
            x[e] = (float)*reinterpret_cast<const _Float16*>(&own[0][0] + place(row, jb + n32));
            if (P == 3) x[e] += (float)*reinterpret_cast<const _Float16*>(&own[0][0] + place_lo(row, jb + n32));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 4; q++) {
            h4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                _Float16 p, r;
                split_hl(g.b * x[4 * q + e] + (g.c / kScaleA) * sum[4 * q + e], p, r);
                hi[e] = p; lo[e] = r;
            }
            const int row = 8 * q + 4 * half + quad, k = jb + (n32 & 28);
            *reinterpret_cast<u2*>(&own[0][0] + place(row, k)) = transpose_quad(__builtin_bit_cast(u2, hi), quad);
            if (P == 3) *reinterpret_cast<u2*>(&own[0][0] + place_lo(row, k)) = transpose_quad(__builtin_bit_cast(u2, lo), quad);
        }
    }
    clear(acc[0]);
    each(std::make_integer_sequence<int, S>{}, [&](auto at_s) __attribute__((always_inline)) {
        constexpr int s = S + decltype(at_s)::value;
        turn(std::integral_constant<int, s>{});   // the first barrier also publishes B
#pragma unroll
        for (int sub = 0; sub < 2; sub++) multiply(own[2 * (s - S) + sub], ring[s % R][sub], wave * 32, acc[0]);
    });
    const int jb = j0 + 32 * wave;
    static_assert(sizeof(ring) >= 4 * 32 * 33 * 4, "the stage of the results fits into the ring");
    float (*out_stage)[33] = reinterpret_cast<float (*)[33]>(&ring[0][0][0] + wave * (32 * 33 * 4));
    if (MODE == kLast) __syncthreads();
    if (jb >= g.w.np) return;
    Addend add;
    load_addend<P, MODE>(g, bt, i0, jb, lane, add);
    finish_block<P, MODE>(g, bt, total(acc[0]), add, i0, jb, lane, false, out_stage);
    if (MODE == kLast) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        write_result(g.out, bt, i0, jb, lane, out_stage);
    }
}

// ---- small matrices: everything in one workgroup -------------------------------------------
// Where X, its transpose and A fit into LDS as operands (64 x 256 with P = 3, 128 x 128 with P = 1),
// all steps run in one launch of one workgroup a matrix: the launches above cost 4 us each, the
// work of one of them here is a fraction of one (all steps, fp32, launches / one workgroup each:
// 1 x 32 x 32 50 / 20 us, 1 x 64 x 64 50 / 25, 1 x 64 x 256 57 / 44, 300 x 64 x 64 91 / 50,
// 1000 x 32 x 128 238 / 94; one product 1 x 128 x 128 50 / 41).  Bound by the chain of five barriers and
// three products a step.  Operands are [32 values][rows][64 bytes] as in
// k_ortho_pair.  A wavefront owns up to two 32 x 32 blocks and keeps their X in fp32 registers
// (C layout: column n32, rows 8 q + 4 half + e), so the a X term needs no lo part.
constexpr int kSmallWaves = 8, kSmallLds = 159 * 1024;
struct SmallArgs {
    InArgs in;
    OutArgs out;
    int mp, np;      // sides rounded up to 32
    int steps;
    float coef[3 * kMaxSteps];
};
template <int P>
constexpr int small_bytes(int mp, int np) { return (2 * mp * np + mp * mp) * (P == 3 ? 4 : 2); }
// byte offset of the hi part of entry (row, k) of an operand of `rows` rows; LO: of its lo part
template <int P, bool LO = false>
__device__ __forceinline__ int place_of(int rows, int row, int k) {
    const int chunk = (P == 3 ? (k & 15) >> 3 : (k & 31) >> 3) + (LO ? 2 : 0);
    return ((P == 3 ? k >> 4 : k >> 5) * rows + row) * 64 + ((chunk ^ ((row >> 2) & 3)) * 16) + (k & 7) * 2;
}
// a block (ib, jb) into the operand whose rows are the block's rows, entry k its column
template <int P>
__device__ __forceinline__ void put_rows_of(unsigned char* m, int rows, int ib, int jb, int lane, const float (&v)[16]) {
    const int n32 = lane & 31, half = lane >> 5, quad = lane & 3;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        h4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            _Float16 p, r;
            split_hl(v[4 * q + e], p, r);
            hi[e] = p; lo[e] = r;
        }
        const int row = ib + 8 * q + 4 * half + quad, k = jb + (n32 & 28);
        *reinterpret_cast<u2*>(m + place_of<P>(rows, row, k)) = transpose_quad(__builtin_bit_cast(u2, hi), quad);
        if (P == 3) *reinterpret_cast<u2*>(m + place_of<P, true>(rows, row, k)) = transpose_quad(__builtin_bit_cast(u2, lo), quad);
    }
}
// ... and whose rows are the block's columns
template <int P>
__device__ __forceinline__ void put_columns_of(unsigned char* m, int rows, int ib, int jb, int lane, const float (&v)[16]) {
    const int n32 = lane & 31, half = lane >> 5;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        h4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            _Float16 p, r;
            split_hl(v[4 * q + e], p, r);
            hi[e] = p; lo[e] = r;
        }
        const int k = ib + 8 * q + 4 * half;
        *reinterpret_cast<h4*>(m + place_of<P>(rows, jb + n32, k)) = hi;
        if (P == 3) *reinterpret_cast<h4*>(m + place_of<P, true>(rows, jb + n32, k)) = lo;
    }
}
// block (ib, jb) of L R^T over `count` times 32 values
template <int P>
__device__ __forceinline__ f16v product_of(const unsigned char* l, int lrows, int ib, const unsigned char* r, int rrows, int jb,
                                           int count, int lane) {
    const int n32 = lane & 31, half = lane >> 5, sw = (n32 >> 2) & 3;
    const unsigned char *lp = l + (ib + n32) * 64, *rp = r + (jb + n32) * 64;
    const int c0 = (half ^ sw) * 16, c1 = ((2 + half) ^ sw) * 16;
    f16v acc[3];
#pragma unroll
    for (int z = 0; z < 3; z++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[z][e] = 0.0f;
#pragma unroll 2
    for (int s = 0; s < count; s++, lp += lrows * 64, rp += rrows * 64) {
        const h8 l0 = *reinterpret_cast<const h8*>(lp + c0), l1 = *reinterpret_cast<const h8*>(lp + c1);
        const h8 r0 = *reinterpret_cast<const h8*>(rp + c0), r1 = *reinterpret_cast<const h8*>(rp + c1);
        acc[0] = mma(l0, r0, acc[0]);
        if (P == 3) {
            acc[1] = mma(l0, r1, acc[1]);
            acc[2] = mma(l1, r0, acc[2]);
        } else {
            acc[1] = mma(l1, r1, acc[1]);
        }
    }
    acc[0] += acc[1];
    if (P == 3) acc[0] += acc[2];
    return acc[0];
}
template <int P>
__global__ __launch_bounds__(64 * kSmallWaves) void k_ortho_small(SmallArgs g) {
    __shared__ __align__(1024) unsigned char lds[kSmallLds];
    __shared__ double ws[kSmallWaves];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n32 = lane & 31, half = lane >> 5;
    const int mp = g.mp, np = g.np, nbi = mp / 32, blocks = nbi * (np / 32), blocks_a = nbi * nbi;
    const int values = P == 3 ? 16 : 32;    // entries in 32 values
    unsigned char* const x_op = lds;                                    // rows of X
    unsigned char* const y_op = x_op + (size_t)mp * np * (P == 3 ? 4 : 2);   // its columns
    unsigned char* const a_op = y_op + (size_t)mp * np * (P == 3 ? 4 : 2);   // A, then B
    const InArgs& in = g.in;
    const OutArgs& o = g.out;
    const size_t bt = blockIdx.x;
    float x[2][16];
    double sum = 0.0;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int id = wave + kSmallWaves * b, ib = id % nbi * 32, jb = id / nbi * 32;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int i = ib + 8 * (e >> 2) + 4 * half + (e & 3), j = jb + n32;
            const int row = o.tall ? j : i, col = o.tall ? i : j;
            x[b][e] = 0.0f;
            if (id < blocks && row < in.rows && col < in.cols) {
                const size_t at_g = bt * in.stride + (size_t)row * in.ld + col;
                float u = load_any(in.g, in.dtype, at_g);
                if (in.mom) {
                    const float m = in.beta * in.mom[at_g] + u;
                    in.mom[at_g] = m;
                    u = in.nesterov ? u + in.beta * m : m;
                }
                if (in.g_clear) in.g_clear[at_g] = 0.0f;
                x[b][e] = u;
                sum += (double)u * (double)u;
            }
        }
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) ws[wave] = sum;
    __syncthreads();
    double squares = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; w++) squares += ws[w];
    const double inv = scale_of(squares, in.eps);
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) x[b][e] = (float)((double)x[b][e] * inv);
#pragma unroll 1
    for (int s = 0; s < g.steps; s++) {
        const float ca = g.coef[3 * s], cb = g.coef[3 * s + 1], cc = g.coef[3 * s + 2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = wave + kSmallWaves * b;
            if (id >= blocks) continue;
            put_rows_of<P>(x_op, mp, id % nbi * 32, id / nbi * 32, lane, x[b]);
            put_columns_of<P>(y_op, np, id % nbi * 32, id / nbi * 32, lane, x[b]);
        }
        __syncthreads();
        float a[2][16];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = wave + kSmallWaves * b, ib = id % nbi * 32, jb = id / nbi * 32;
            if (id >= blocks_a) continue;
            const f16v p = product_of<P>(x_op, mp, ib, x_op, mp, jb, np / values, lane);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                a[b][e] = p[e] * (kScaleA / (kScaleX * kScaleX));
                // one product: b A takes the A that A A is made of, so that their errors go together
                if (P == 1) a[b][e] = (float)(_Float16)a[b][e];
            }
            put_rows_of<P>(a_op, mp, ib, jb, lane, a[b]);
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = wave + kSmallWaves * b, ib = id % nbi * 32, jb = id / nbi * 32;
            if (id >= blocks_a) continue;
            const f16v p = product_of<P>(a_op, mp, ib, a_op, mp, jb, mp / values, lane);
#pragma unroll
            for (int e = 0; e < 16; e++) a[b][e] = cb * a[b][e] + (cc / kScaleA) * p[e];
        }
        __syncthreads();   // A is read
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = wave + kSmallWaves * b;
            if (id < blocks_a) put_rows_of<P>(a_op, mp, id % nbi * 32, id / nbi * 32, lane, a[b]);
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = wave + kSmallWaves * b;
            if (id >= blocks) continue;
            const f16v p = product_of<P>(a_op, mp, id % nbi * 32, y_op, np, id / nbi * 32, mp / values, lane);
#pragma unroll
            for (int e = 0; e < 16; e++) x[b][e] = ca * x[b][e] + p[e] * (1.0f / kScaleA);
        }
        __syncthreads();   // X transposed and B are read
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int id = wave + kSmallWaves * b, ib = id % nbi * 32, jb = id / nbi * 32;
        if (id >= blocks) continue;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int i = ib + 8 * (e >> 2) + 4 * half + (e & 3), j = jb + n32;
            const int row = o.tall ? j : i, col = o.tall ? i : j;
            if (row < o.rows && col < o.cols) put_out(o, bt * o.stride + (size_t)row * o.ld + col, x[b][e] * (1.0f / kScaleX));
        }
    }
}

// steps = 0: the scaled input itself
template <int P>
__global__ __launch_bounds__(256) void k_ortho_copy(Work w, OutArgs t) {
    const int64_t total = (int64_t)t.rows * t.cols;
    const size_t bt = blockIdx.y;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int r = (int)(e / t.cols), c = (int)(e - (int64_t)r * t.cols);
        const int j = t.tall ? r : c, i = t.tall ? c : r;
        const _Float16* y = w.y[0] + bt * w.np * (size_t)w.ldm;
        const size_t o = at<P>(j, w.ldm, i);
        const float v = (float)y[o] + (float)(P == 3 ? y[o + kLo] : w.y_lo[bt * w.np * (size_t)w.ldm + o]);
        put_out(t, bt * t.stride + (size_t)r * t.ld + c, v * (1.0f / kScaleX));
    }
}

// ---- plan ------------------------------------------------------------------------------
struct Plan {
    int mp, np, ldm, ldn, groups;
    int splits;   // of X X^T
    bool small;   // k_ortho_small
    size_t part, x, y, y_lo, ab, split_part, total;   // bytes
};
constexpr int kOverhang = 256 - 64;
size_t round_up(size_t v, size_t q) { return (v + q - 1) / q * q; }
// Tile size of a product: rounds of 256 workgroups (one a CU) times what a tile costs relative to
// a 64 x 64 one.  A tile twice as wide does four times the work in 2.1 times the time: it reads
// half as much from L2 and LDS an operation.  Measured at 4096 x 4096, P = 1: B X on tiles of
// 256 / 192 / 128: 138 / 152 / 151 us; X X^T (253 tiles of 192 fill the machine, 136 of 256 half of
// it): 82 / 70 / 90 us.  At 1000 x 2731, P = 3: B X on 192 / 128 / 64: 41 / 26 / 29 us, X X^T on
// 128 / 64: 40 / 19 us.
int tile_for(bool sym, int rows, int cols, int batch) {
    constexpr float cost[5] = {0.0f, 1.0f, 2.1f, 4.3f, 7.5f};
    int best = 1;
    float least = 0.0f;
    for (int f = 1; f <= 4; f++) {
        const int64_t ti = (rows + 64 * f - 1) / (64 * f), tj = (cols + 64 * f - 1) / (64 * f);
        const int64_t tiles = (sym ? ti * (ti + 1) / 2 : ti * tj) * batch;
        const float c = (float)((tiles + 255) / 256) * cost[f];
        if (f == 1 || c < least) { least = c; best = f; }
    }
    return best;
}
// k_ortho_block while its blocks find a CU each (two or four: 700 x 700 fp32, all steps, 130 us
// instead of 120) and a wavefront's share of the K axis is short (of 126 stages: 250 x 2000 fp32
// 124 us, split over workgroups 118; of 63: with one product 91 us, split 99)
bool in_blocks(bool sym, int rows, int cols, int batch, int stages) {
    const int64_t ti = rows / 32, tj = cols / 32;
    return (sym ? ti * (ti + 1) / 2 : ti * tj) * batch <= 256 && stages <= 100;
}
Plan make_plan(int batch, int rows, int cols, int products) {
    Plan p{};
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    p.mp = (int)round_up(m, 32);
    p.np = (int)round_up(n, 32);
    p.small = p.mp <= 1024 && p.np <= 1024 && p.mp * p.np <= 2 * kSmallWaves * 1024 &&
              (products == 3 ? small_bytes<3>(p.mp, p.np) : small_bytes<1>(p.mp, p.np)) <= kSmallLds;
    if (p.small) return p;   // no workspace
    p.mp = (int)round_up(m, 64);
    p.np = (int)round_up(n, 64);
    const int planes = products == 3 ? 2 : 1;
    p.ldm = p.mp * planes;
    p.ldn = p.np * planes;
    const size_t h = sizeof(_Float16);
    // a wavefront of the first pass takes two or more pieces of 256 columns
    const int64_t units = (int64_t)rows * ((cols + 255) / 256);
    p.groups = (int)(units / 8 < 1 ? 1 : units / 8 > kMaxNormGroups ? kMaxNormGroups : units / 8);
    p.part = round_up((size_t)batch * p.groups * sizeof(double), 256);
    // A tile that hangs over the last row of a batch reads up to kOverhang rows behind it: into
    // the next matrix or this slack.  What it reads there reaches only rows that are not stored.
    p.x = round_up(((size_t)batch * p.mp + kOverhang) * p.ldn * h, 256);
    p.y = round_up(((size_t)batch * p.np + kOverhang) * p.ldm * h, 256);
    p.y_lo = products == 1 ? round_up((size_t)batch * p.np * p.ldm * h, 256) : 0;
    p.ab = round_up(((size_t)batch * p.mp + kOverhang) * p.ldm * h, 256);
    // X X^T of few small tiles with many stages: the stages shared out until about two workgroups a
    // CU run, none with less than 16 stages of 64 values (all steps, fp32, unsplit / 8 / 16 / 32 stages:
    // 1 x 64 x 2048: 101 / 75 / 78 / 88 us, 1 x 250 x 4000: 200 / 139 / 136 / 149,
    // 1 x 500 x 4500: 264 / 215 / 213 / 199; 1 x 250 x 1000, one product: 80 / 86 / 80 / 80).  Two workgroups
    // a tile on half of the CUs gain nothing (1 x 1000 x 2731, one product: 200 us unsplit, 219 split).
    p.splits = 1;
    if (tile_for(true, p.mp, p.mp, batch) == 1 && !in_blocks(true, p.mp, p.mp, batch, p.ldn / 32)) {
        const int64_t nt = p.mp / 64, tiles = nt * (nt + 1) / 2 * batch;
        const int64_t room = 512 / tiles, most = p.ldn / 64 / 16;
        const int64_t splits = tiles > 128 ? 1 : room < most ? room : most;
        p.splits = (int)(splits < 1 ? 1 : splits > 16 ? 16 : splits);
        if (p.splits > 1) p.split_part = (size_t)tiles * p.splits * 64 * 64 * sizeof(float);
    }
    p.total = p.part + p.x + 2 * p.y + p.y_lo + 2 * p.ab + p.split_part;
    return p;
}

// An XCD takes whole matrices while their tiles find a CU each there (32 of them): its L2 fetches
// its own matrices only (9 x 256 x 256 fp32, all steps: 93 us instead of 109).
bool one_xcd_each(int batch, int64_t tiles) { return batch >= 8 && tiles * ((batch + 7) / 8) <= 32; }

template <int P, int MODE, int F, int SUB, int R>
void run_mul(MulArgs g, int batch, hipStream_t st) {
    constexpr int T = 64 * F;
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    g.tiles_i = (g.w.mp + T - 1) / T;
    const int tiles_j = (g.w.np + T - 1) / T;
    const int tiles = g.tiles = SYM ? g.tiles_i * (g.tiles_i + 1) / 2 : g.tiles_i * tiles_j;
    const int per_xcd = (batch + 7) / 8;
    g.by_xcd = one_xcd_each(batch, tiles) ? batch : 0;
    // Workgroups go to the eight XCDs in turn.  Where the CUs take more than one each, an XCD takes a
    // run of tiles of neighbouring rows and columns, which share panels in its L2; one tile a CU is
    // faster in plain order, where an XCD keeps to one row's panel (all steps, runs / plain order:
    // 2048 x 8192 one product 998 / 1030 us, 1000 x 2731 fp32 292 / 302; 2 x 500 x 1000 fp32 160 / 135,
    // 700 x 700 fp32 138 / 124).
    g.runs = !g.by_xcd && (int64_t)tiles * F * batch > 256;
    g.row_len = SYM ? g.tiles_i + 1 : g.runs ? 4 * tiles_j : g.tiles_i;
    g.row_inv = (((uint64_t)1 << 32) + g.row_len - 1) / g.row_len;
    hipLaunchKernelGGL((k_ortho_mul<P, MODE, F, SUB, R>), dim3(g.by_xcd ? 8 * tiles : tiles, g.by_xcd ? per_xcd : batch, MODE == kGram && F == 1 ? g.splits : 1), dim3(256),
                       0, st, g);
    if (MODE == kGram && F == 1 && g.splits > 1) hipLaunchKernelGGL(k_ortho_fold<P>, dim3(tiles, batch), dim3(256), 0, st, g);
}
template <int P, int MODE>
void run_block(MulArgs g, int batch, hipStream_t st) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    g.tiles_i = g.w.mp / 32;
    const int tiles_j = g.w.np / 32, tiles = g.tiles = SYM ? g.tiles_i * (g.tiles_i + 1) / 2 : g.tiles_i * tiles_j;
    g.by_xcd = one_xcd_each(batch, tiles) ? batch : 0;
    g.row_len = SYM ? g.tiles_i + 1 : g.tiles_i;
    g.row_inv = (((uint64_t)1 << 32) + g.row_len - 1) / g.row_len;
    hipLaunchKernelGGL((k_ortho_block<P, MODE>), dim3(g.by_xcd ? 8 * tiles : tiles, g.by_xcd ? (batch + 7) / 8 : batch), dim3(64 * kBlockWaves), 0, st, g);
}
// Ring buffers: three to four stages in flight where they fit into 160 KiB (with two, a stage of
// small tiles is over before the copies of the next have landed: 42 instead of 19 us above); tiles
// of 128 with P = 1 run faster as two workgroups a CU of two stages each.
template <int P, int MODE>
void run_mul(const MulArgs& g, int batch, hipStream_t st) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    if (in_blocks(SYM, g.w.mp, SYM ? g.w.mp : g.w.np, batch, g.stages)) { run_block<P, MODE>(g, batch, st); return; }
    switch (tile_for(SYM, g.w.mp, SYM ? g.w.mp : g.w.np, batch)) {
        case 4: run_mul<P, MODE, 4, P == 1 ? 1 : 2, P == 1 ? 4 : 2>(g, batch, st); break;
        case 3: run_mul<P, MODE, 3, 2, 3>(g, batch, st); break;
        case 2: run_mul<P, MODE, 2, 2, P == 1 ? 2 : 4>(g, batch, st); break;
        default: run_mul<P, MODE, 1, 2, 4>(g, batch, st); break;
    }
}

// The pair kernel reads all of A in every workgroup: worth it up to 128 KiB of A (m = 128 with
// P = 3, 256 with P = 1) and while one or two rounds of workgroups do.  All five steps, with it and
// without: 1 x 128 x 512 fp32 68 / 80 us, 1 x 192 x 800 fp32 95 / 95, 1 x 256 x 843 fp32 114 / 104,
// the same with one product 78 / 84.
template <int P>
bool use_pair(const Work& w, int batch) {
    return w.mp <= (P == 3 ? 128 : 256) && (int64_t)(w.mp / 32) * ((w.np + 127) / 128) * batch <= 512;
}
template <int P, int MODE>
void run_pair(MulArgs g, int batch, hipStream_t st) {
    const int ti = g.w.mp / 32, tj = (g.w.np + 127) / 128, per_xcd = (batch + 7) / 8;
    g.by_xcd = one_xcd_each(batch, ti * tj) ? batch : 0;
    const dim3 grid(g.by_xcd ? 8 * ti : ti, tj, g.by_xcd ? per_xcd : batch), block(256);
    switch (g.w.mp / 64) {
        case 1: hipLaunchKernelGGL((k_ortho_pair<P, MODE, 1>), grid, block, 0, st, g); break;
        case 2: hipLaunchKernelGGL((k_ortho_pair<P, MODE, 2>), grid, block, 0, st, g); break;
        case 3: if constexpr (P == 1) hipLaunchKernelGGL((k_ortho_pair<P, MODE, 3>), grid, block, 0, st, g); break;
        default: if constexpr (P == 1) hipLaunchKernelGGL((k_ortho_pair<P, MODE, 4>), grid, block, 0, st, g); break;
    }
}

template <int P>
int run_all(const InArgs& in, const OutArgs& out, int batch, int steps, const float* coef, const Plan& p, char* work,
            hipStream_t st) {
    if (p.small) {
        SmallArgs g{};
        g.in = in; g.out = out; g.mp = p.mp; g.np = p.np; g.steps = steps;
        for (int i = 0; i < 3 * steps; i++) g.coef[i] = coef[i];
        hipLaunchKernelGGL(k_ortho_small<P>, dim3(batch), dim3(64 * kSmallWaves), 0, st, g);
        CFP_HIP_TRY(hipGetLastError());
        return 0;
    }
    Work w{};
    InArgs a = in;
    a.part = (double*)work;             work += p.part;
    a.groups = p.groups;
    a.vec = a.cols % 4 == 0 && a.ld % 4 == 0 && a.stride % 4 == 0 &&
            (reinterpret_cast<uintptr_t>(a.g) & (a.dtype == CFP_F32 ? 15u : 7u)) == 0 &&
            (reinterpret_cast<uintptr_t>(a.mom) & 15u) == 0;
    w.x = (_Float16*)work;              work += p.x;
    w.y[0] = (_Float16*)work;           work += p.y;
    w.y[1] = (_Float16*)work;           work += p.y;
    w.y_lo = P == 1 ? (_Float16*)work : nullptr; work += p.y_lo;
    w.a = (_Float16*)work;              work += p.ab;
    w.b = (_Float16*)work;              work += p.ab;
    f4* split_part = (f4*)work;
    w.mp = p.mp; w.np = p.np; w.ldm = p.ldm; w.ldn = p.ldn;
    const int tall = out.tall;
    hipLaunchKernelGGL(k_ortho_norm, dim3(p.groups, batch), dim3(256), 0, st, a);
    const int rp = tall ? p.np : p.mp, cp = tall ? p.mp : p.np;
    hipLaunchKernelGGL(k_ortho_load<P>, dim3(cp / 64, rp / 64, batch), dim3(256), 0, st, a, w, tall);
    if (steps == 0) {
        const int64_t g = ((int64_t)out.rows * out.cols + 255) / 256;
        hipLaunchKernelGGL(k_ortho_copy<P>, dim3((unsigned)(g < 4096 ? g : 4096), batch), dim3(256), 0, st, w, out);
    }
    const size_t xb = (size_t)p.mp * p.ldn, yb = (size_t)p.np * p.ldm, ab = (size_t)p.mp * p.ldm;
    for (int s = 0; s < steps; s++) {
        MulArgs g{};
        g.w = w;
        g.cur = s & 1;
        g.a = coef[3 * s]; g.b = coef[3 * s + 1]; g.c = coef[3 * s + 2];
        g.out = out;
        g.l = g.r = w.x; g.ldl = g.ldr = p.ldn; g.l_batch = g.r_batch = xb; g.stages = p.ldn / 32;
        g.splits = p.splits; g.part = split_part;
        run_mul<P, kGram>(g, batch, st);
        if (use_pair<P>(w, batch)) {
            if (s + 1 < steps) run_pair<P, kStep>(g, batch, st);
            else run_pair<P, kLast>(g, batch, st);
            continue;
        }
        g.l = g.r = w.a; g.ldl = g.ldr = p.ldm; g.l_batch = g.r_batch = ab; g.stages = p.ldm / 32;
        run_mul<P, kPoly>(g, batch, st);
        g.l = w.b; g.r = w.y[g.cur]; g.ldl = g.ldr = p.ldm; g.l_batch = ab; g.r_batch = yb; g.stages = p.ldm / 32;
        if (s + 1 < steps) run_mul<P, kStep>(g, batch, st);
        else run_mul<P, kLast>(g, batch, st);
    }
    CFP_HIP_TRY(hipGetLastError());
    return 0;
}

// the quintic of the Muon optimiser's write-up (K. Jordan, 2024): slope 3.44 at zero, singular
// values in 0.7 .. 1.2 after five steps
constexpr float kQuintic[3] = {3.4445f, -4.7750f, 2.0315f};
constexpr int kMaxSide = 1 << 16;

int check_sizes(const char* who, int batch, int rows, int cols, int steps, int products, float eps) {
    CFP_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 1 && cols >= 1 && rows <= kMaxSide && cols <= kMaxSide,
                "%s: batch must be in 0..65535 and rows and cols in 1..65536 (got %d, %d, %d)", who, batch, rows, cols);
    CFP_REQUIRE(steps >= 0 && steps <= kMaxSteps, "%s: steps must be in 0..%d (got %d)", who, kMaxSteps, steps);
    CFP_REQUIRE(products == 0 || products == 1 || products == 3, "%s: products must be 0 (by type), 1 or 3 (got %d)", who, products);
    CFP_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", who);
    return 0;
}
void fill_coef(const float* coefs, int steps, float (&c)[3 * kMaxSteps]) {
    for (int i = 0; i < 3 * steps; i++) c[i] = coefs ? coefs[i] : kQuintic[i % 3];
}
size_t type_bytes(int dtype) { return dtype == CFP_F32 ? 4 : 2; }

}  // namespace
}  // namespace cfp

using namespace cfp;

extern "C" {

size_t cfp_orthogonalize_workspace(int batch, int rows, int cols, int products) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || rows > kMaxSide || cols > kMaxSide || (products != 1 && products != 3))
        return 0;
    return make_plan(batch, rows, cols, products).total;
}

int cfp_orthogonalize(const void* d_g, int dtype, int64_t ld, int64_t batch_stride, int batch, int rows, int cols,
                      int steps, const float* coefs, float eps, int products, void* d_out, int64_t ld_out,
                      int64_t out_batch_stride, void* d_work, size_t work_bytes, void* stream) {
    CFP_REQUIRE(dtype == CFP_F32 || dtype == CFP_BF16 || dtype == CFP_F16,
                "cfp_orthogonalize: dtype must be CFP_F32, CFP_BF16 or CFP_F16 (got %d)", dtype);
    if (check_sizes("cfp_orthogonalize", batch, rows, cols, steps, products, eps)) return 1;
    if (batch == 0) return 0;
    CFP_REQUIRE(d_g && d_out, "cfp_orthogonalize: NULL input or output");
    CFP_REQUIRE((ld >= cols || rows == 1) && (ld_out >= cols || rows == 1) && ld >= 0 && ld_out >= 0,
                "cfp_orthogonalize: rows of %d need strides of at least that (got %lld, %lld)", cols, (long long)ld,
                (long long)ld_out);
    const int64_t span = (int64_t)(rows - 1) * ld + cols, span_out = (int64_t)(rows - 1) * ld_out + cols;
    CFP_REQUIRE(batch == 1 || (batch_stride >= span && out_batch_stride >= span_out),
                "cfp_orthogonalize: matrices of a batch must not overlap (strides %lld, %lld)", (long long)batch_stride,
                (long long)out_batch_stride);
    const unsigned am = (unsigned)type_bytes(dtype) - 1u;
    CFP_REQUIRE(((reinterpret_cast<uintptr_t>(d_g) | reinterpret_cast<uintptr_t>(d_out)) & am) == 0,
                "cfp_orthogonalize: input or output not aligned to its type");
    CFP_REQUIRE((d_g == d_out && (ld == ld_out || rows == 1) && (batch_stride == out_batch_stride || batch == 1)) ||
                    apart(d_g, ld, batch_stride, d_out, ld_out, out_batch_stride, batch, rows, cols, type_bytes(dtype)),
                "cfp_orthogonalize: the output may replace the input, with the same strides, but not overlap it otherwise");
    const int p = products ? products : 3;
    const Plan plan = make_plan(batch, rows, cols, p);
    CFP_REQUIRE(plan.total == 0 || (d_work && work_bytes >= plan.total && (reinterpret_cast<uintptr_t>(d_work) & 255u) == 0),
                "cfp_orthogonalize: needs a 256-byte aligned workspace of %zu bytes (got %zu)", plan.total, work_bytes);
    float c[3 * kMaxSteps];
    fill_coef(coefs, steps, c);
    InArgs in{};
    in.g = d_g; in.dtype = dtype; in.ld = ld; in.stride = batch > 1 ? batch_stride : 0; in.rows = rows; in.cols = cols; in.eps = eps;
    OutArgs out{};
    out.out = d_out; out.dtype = dtype; out.ld = ld_out; out.stride = out_batch_stride;
    out.rows = rows; out.cols = cols; out.tall = rows > cols;
    return p == 3 ? run_all<3>(in, out, batch, steps, c, plan, (char*)d_work, (hipStream_t)stream)
                  : run_all<1>(in, out, batch, steps, c, plan, (char*)d_work, (hipStream_t)stream);
}

}  // extern "C"

namespace cfp {

int muon_update(const MuonArgs& u, hipStream_t st) {
    if (check_sizes("cfp_muon_update", u.batch, u.rows, u.cols, u.steps, u.products, u.eps)) return 1;
    CFP_REQUIRE(u.scale >= 0.0f, "cfp_muon_update: scale must not be negative (got %g)", (double)u.scale);
    if (u.batch == 0) return 0;
    CFP_REQUIRE(u.w && u.g && u.mom, "cfp_muon_update: NULL weight, gradient or momentum");
    CFP_REQUIRE(u.ld >= u.cols || (u.rows == 1 && u.ld >= 0), "cfp_muon_update: rows of %d need a stride of at least that (got %lld)",
                u.cols, (long long)u.ld);
    CFP_REQUIRE(u.batch == 1 || u.stride >= (int64_t)(u.rows - 1) * u.ld + u.cols,
                "cfp_muon_update: matrices of a batch must not overlap (stride %lld)", (long long)u.stride);
    CFP_REQUIRE(((reinterpret_cast<uintptr_t>(u.w) | reinterpret_cast<uintptr_t>(u.g) | reinterpret_cast<uintptr_t>(u.mom)) & 3u) == 0,
                "cfp_muon_update: arrays not aligned to fp32");
    const int p = u.products ? u.products : 3;
    const Plan plan = make_plan(u.batch, u.rows, u.cols, p);
    CFP_REQUIRE(plan.total == 0 || (u.work && u.work_bytes >= plan.total && (reinterpret_cast<uintptr_t>(u.work) & 255u) == 0),
                "cfp_muon_update: needs a 256-byte aligned workspace of %zu bytes (got %zu)", plan.total, u.work_bytes);
    for (const float* pair : {u.g, u.mom})
        CFP_REQUIRE(apart(u.w, u.ld, u.stride, pair, u.ld, u.stride, u.batch, u.rows, u.cols, 4),
                    "cfp_muon_update: weight, gradient and momentum must not overlap");
    CFP_REQUIRE(apart(u.g, u.ld, u.stride, u.mom, u.ld, u.stride, u.batch, u.rows, u.cols, 4),
                "cfp_muon_update: weight, gradient and momentum must not overlap");
    float c[3 * kMaxSteps];
    fill_coef(u.coefs, u.steps, c);
    InArgs in{};
    in.g = u.g; in.dtype = CFP_F32; in.ld = u.ld; in.stride = u.batch > 1 ? u.stride : 0; in.rows = u.rows; in.cols = u.cols;
    in.mom = u.mom; in.beta = u.beta; in.nesterov = u.nesterov; in.eps = u.eps;
    in.g_clear = u.clear_g ? u.g : nullptr;
    OutArgs out{};
    out.out = u.w; out.dtype = CFP_F32; out.ld = u.ld; out.stride = u.stride;
    out.rows = u.rows; out.cols = u.cols; out.tall = u.rows > u.cols;
    out.update = 1; out.lr_dev = u.lr_dev; out.lr = u.lr; out.decay = u.decay;
    // 0: sqrt(outputs / inputs) where that is above 1, of a weight [outputs][inputs]
    out.scale = u.scale > 0.0f ? u.scale : u.rows > u.cols ? sqrtf((float)u.rows / (float)u.cols) : 1.0f;
    return p == 3 ? run_all<3>(in, out, u.batch, u.steps, c, plan, (char*)u.work, st)
                  : run_all<1>(in, out, u.batch, u.steps, c, plan, (char*)u.work, st);
}

}  // namespace cfp

extern "C" int cfp_muon_update(float* d_w, const float* d_g, float* d_momentum, int64_t ld, int64_t batch_stride,
                               int batch, int rows, int cols, const float* d_lr, float lr, float momentum,
                               int nesterov, float weight_decay, float scale, int steps, const float* coefs,
                               float eps, int products, void* d_work, size_t work_bytes, void* stream) {
    MuonArgs u{};
    u.w = d_w; u.g = const_cast<float*>(d_g); u.mom = d_momentum; u.ld = ld; u.stride = batch_stride;
    u.batch = batch; u.rows = rows; u.cols = cols; u.lr_dev = d_lr; u.lr = lr; u.beta = momentum;
    u.nesterov = nesterov; u.decay = weight_decay; u.scale = scale; u.steps = steps; u.coefs = coefs;
    u.eps = eps; u.products = products; u.work = d_work; u.work_bytes = work_bytes; u.clear_g = 0;
    return muon_update(u, (hipStream_t)stream);
}
