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
//   P = 3  every matrix is a pair hi + lo of fp16 numbers (22 bits, or to 2^-35 of 1) and a
//          product is hi hi + hi lo + lo hi: what is left out, lo lo, is below 2^-22 of a
//          product.  Error against 64 bits about 1e-6 of the result's norm, as fp32 has.
//          For fp32 and fp16 inputs.
//   P = 1  one fp16 product; X alone keeps its lo part, for the term a X.  Without it the
//          rounding of X at every step is amplified by a (3.44) a step where singular values
//          are small: 5e-3 of the norm measured instead of 1 to 2e-3, which is a bf16 rounding
//          (1.7e-3).  A third of the matrix instructions.  For bf16 inputs.
#include <float.h>

#include "cfp_internal.h"

namespace cfp {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr float kScaleX = 1024.0f, kScaleA = 256.0f;
constexpr int kMaxSteps = 16;
constexpr int kNormGroups = 64;   // partial sums of squares a matrix

// A row of a P = 3 matrix: blocks of 32 entries, the 32 hi parts then the 32 lo parts, so that
// the 64 values of one LDS stage are one contiguous 128-byte piece either way.
template <int P>
__device__ __forceinline__ size_t at(size_t row, int ld, int k) {
    return row * ld + (P == 3 ? (k >> 5) * 64 + (k & 31) : k);
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
    float* mom;          // or null; same ld and stride as g
    float beta;
    int nesterov;
    float* g_clear;      // or null: zeroed behind its last read
    double* part;        // [batch][kNormGroups]
    float eps;
};
__device__ __forceinline__ float load_any(const void* p, int dtype, size_t i) {
    return dtype == CFP_F32 ? ((const float*)p)[i]
                            : dtype == CFP_BF16 ? (float)((const __bf16*)p)[i] : (float)((const _Float16*)p)[i];
}

// First pass: momentum and the sum of squares (64 bits: squares of fp32 values neither
// overflow nor vanish).
__global__ __launch_bounds__(256) void k_ortho_norm(InArgs a) {
    __shared__ double ws[4];
    const size_t base = (size_t)blockIdx.y * a.stride;
    double s = 0.0;
    const int64_t total = (int64_t)a.rows * a.cols;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)kNormGroups * 256) {
        const int r = (int)(e / a.cols), c = (int)(e - (int64_t)r * a.cols);
        const size_t i = base + (size_t)r * a.ld + c;
        float u = load_any(a.g, a.dtype, i);
        if (a.mom) {
            const float m = a.beta * a.mom[i] + u;
            a.mom[i] = m;
            u = a.nesterov ? u + a.beta * m : m;
        }
        s += (double)u * (double)u;
    }
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[(size_t)blockIdx.y * kNormGroups + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// The matrices of one call.  All live in the workspace, padded with zeros to whole tiles, which
// the products keep zero; no kernel below needs a bounds check but the last store.
struct Work {
    _Float16* x;        // [batch][mp][ldn]   X
    _Float16* y[2];     // [batch][np][ldm]   X transposed, before and after a step
    _Float16* y_lo;     // [batch][np][mp]    P = 1: what X transposed lost in its rounding
    _Float16* a;        // [batch][mp][ldm]
    _Float16* b;        // [batch][mp][ldm]
    int mp, np, ldm, ldn;
};

// Second pass: X = u / (|u| + eps) times kScaleX in both orders, zeros in the padding.
template <int P>
__global__ __launch_bounds__(256) void k_ortho_load(InArgs a, Work w, int tall) {
    __shared__ float tile[64][65];
    __shared__ float inv_s;
    const int bt = blockIdx.z;
    if (threadIdx.x < 64) {
        static_assert(kNormGroups == 64, "one partial sum a lane");
        double s = a.part[(size_t)bt * kNormGroups + threadIdx.x];
        for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
        if (threadIdx.x == 0) inv_s = (float)((double)kScaleX / (sqrt(s) + (double)a.eps));
    }
    __syncthreads();
    const float inv = inv_s;
    const size_t base = (size_t)bt * a.stride;
    // G's rows and columns, padded
    const int r0 = (int)blockIdx.y * 64, c0 = (int)blockIdx.x * 64;
    _Float16* d1 = tall ? w.y[0] + (size_t)bt * w.np * w.ldm : w.x + (size_t)bt * w.mp * w.ldn;
    _Float16* d2 = tall ? w.x + (size_t)bt * w.mp * w.ldn : w.y[0] + (size_t)bt * w.np * w.ldm;
    const int ld1 = tall ? w.ldm : w.ldn, ld2 = tall ? w.ldn : w.ldm;
    _Float16* lo = P == 1 ? w.y_lo + (size_t)bt * w.np * w.mp : nullptr;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const int r = r0 + i, c = c0 + tx;
        float u = 0.0f;
        if (r < a.rows && c < a.cols) {
            const size_t o = base + (size_t)r * a.ld + c;
            u = load_any(a.g, a.dtype, o);
            if (a.g_clear) a.g_clear[o] = 0.0f;
            if (a.mom) {
                const float m = a.mom[o];
                u = a.nesterov ? u + a.beta * m : m;
            }
            u *= inv;
        }
        tile[i][tx] = u;
        _Float16 hi, lw;
        split_hl(u, hi, lw);
        const size_t o = at<P>(r, ld1, c);
        d1[o] = hi;
        if (P == 3) d1[o + 32] = lw;
        if (P == 1 && tall) lo[(size_t)r * w.mp + c] = lw;
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        _Float16 hi, lw;
        split_hl(tile[tx][i], hi, lw);
        const size_t o = at<P>(c0 + i, ld2, r0 + tx);
        d2[o] = hi;
        if (P == 3) d2[o + 32] = lw;
        if (P == 1 && !tall) lo[(size_t)(c0 + i) * w.mp + r0 + tx] = lw;
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

// ---- the product C[i][j] = sum_k L[i][k] R[j][k] and what is made of it ---------------
enum { kGram, kPoly, kStep, kLast };
struct MulArgs {
    const _Float16* l;
    const _Float16* r;
    int ldl, ldr;            // values (hi and lo counted apart) a row
    size_t l_batch, r_batch; // values a matrix
    int stages;              // of 64 values
    int tiles_i, tiles_j;
    Work w;
    int cur;                 // y[cur] is X transposed before the step
    float a, b, c;
    OutArgs out;
};
__device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// WM x WN wavefronts of FM x FN blocks of 32 x 32.  A stage is 64 values of every row of the
// tile's L and R sides, 128 bytes a row, copied to LDS without registers (each lane's 16 bytes
// land at the wave's base + 16 * lane) one stage ahead.  16-byte chunk c of row r sits at chunk
// c ^ (r & 7): eight consecutive rows' fragments then cover all banks.
template <int P, int MODE, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(64 * WM * WN) void k_ortho_mul(MulArgs g) {
    constexpr int TM = 32 * WM * FM, TN = 32 * WN * FN, WAVES = WM * WN;
    constexpr int LOADS = (TM + TN) / 8 / WAVES;   // 1 KiB pieces (8 rows) a wave
    static_assert((TM / 8) % WAVES == 0 && (TN / 8) % WAVES == 0, "whole pieces a wave on either side");
    __shared__ __align__(1024) unsigned char lds[2][(TM + TN) * 128];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n32 = lane & 31, half = lane >> 5;
    int ti, tj;
    if (MODE == kGram || MODE == kPoly) {   // tiles on and above the diagonal, by columns
        int t = (int)blockIdx.x;
        tj = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while ((tj + 1) * (tj + 2) / 2 <= t) tj++;
        while (tj * (tj + 1) / 2 > t) tj--;
        ti = t - tj * (tj + 1) / 2;
    } else {
        ti = (int)blockIdx.x % g.tiles_i;
        tj = (int)blockIdx.x / g.tiles_i;
    }
    const size_t bt = blockIdx.y;
    const int i0 = ti * TM, j0 = tj * TN;
    const _Float16* lsrc = g.l + bt * g.l_batch + (size_t)i0 * g.ldl;
    const _Float16* rsrc = g.r + bt * g.r_batch + (size_t)j0 * g.ldr;

    const int prow = lane >> 3, pchunk = (lane & 7) ^ (prow & 7);
    auto copy_stage = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < LOADS; q++) {
            constexpr int LL = TM / 8 / WAVES;   // the first LL pieces are of the L side
            const int piece = (q < LL ? q : q - LL) * WAVES + wave;
            const _Float16* src = q < LL ? lsrc : rsrc;
            const int ld = q < LL ? g.ldl : g.ldr;
            const _Float16* from = src + (size_t)piece * 8 * ld + (size_t)s * 64;   // uniform
            const unsigned voff = (unsigned)(prow * ld * 2 + pchunk * 16);
            const unsigned to = (unsigned)(size_t)&lds[buf][((q < LL ? 0 : TM) + piece * 8) * 128];
            asm volatile(
                "s_mov_b32 m0, %2\n\t"
                "s_nop 0\n\t"
                "global_load_lds_dwordx4 %0, %1"
                :
                : "v"(voff), "s"(from), "s"(to)
                : "memory", "m0");
        }
    };

    f16v acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    const int wi = (wave % WM) * FM * 32, wj = (wave / WM) * FN * 32;
    auto frag = [&](int buf, int row, int chunk) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(&lds[buf][row * 128 + ((chunk ^ (row & 7)) * 16)]);
    };
    copy_stage(0, 0);
    for (int s = 0; s < g.stages; s++) {
        // this wave's pieces of stage s have landed; behind the barrier everyone's have, and
        // nobody reads the other buffer any more
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const int buf = s & 1;
        if (s + 1 < g.stages) copy_stage(s + 1, buf ^ 1);
        if (P == 1) {
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                h8 l[FM], r[FN];
#pragma unroll
                for (int i = 0; i < FM; i++) l[i] = frag(buf, wi + 32 * i + n32, 2 * ks + half);
#pragma unroll
                for (int j = 0; j < FN; j++) r[j] = frag(buf, TM + wj + 32 * j + n32, 2 * ks + half);
#pragma unroll
                for (int i = 0; i < FM; i++)
#pragma unroll
                    for (int j = 0; j < FN; j++) acc[i][j] = mma(l[i], r[j], acc[i][j]);
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                h8 l[2][FM], r[2][FN];
#pragma unroll
                for (int z = 0; z < 2; z++) {
#pragma unroll
                    for (int i = 0; i < FM; i++) l[z][i] = frag(buf, wi + 32 * i + n32, 4 * z + 2 * ks + half);
#pragma unroll
                    for (int j = 0; j < FN; j++) r[z][j] = frag(buf, TM + wj + 32 * j + n32, 4 * z + 2 * ks + half);
                }
#pragma unroll
                for (int z = 0; z < 3; z++)   // hi hi, hi lo, lo hi
#pragma unroll
                    for (int i = 0; i < FM; i++)
#pragma unroll
                        for (int j = 0; j < FN; j++)
                            acc[i][j] = mma(l[z == 2][i], r[z == 1][j], acc[i][j]);
            }
        }
    }

    // Lane's part of a block: column n32, rows 8 q + 4 half + 0..3 (q = 0..3), so four
    // consecutive entries of a row of the transposed matrix.
#pragma unroll
    for (int fi = 0; fi < FM; fi++)
#pragma unroll
        for (int fj = 0; fj < FN; fj++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int i = i0 + wi + 32 * fi + 8 * q + 4 * half, j = j0 + wj + 32 * fj + n32;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[fi][fj][4 * q + e];
                if (MODE == kGram || MODE == kPoly) {
                    _Float16* m = (MODE == kGram ? g.w.a : g.w.b) + bt * g.w.mp * (size_t)g.w.ldm;
                    const size_t across = at<P>(j, g.w.ldm, i);
                    if (MODE == kGram) {
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] *= kScaleA / (kScaleX * kScaleX);
                    } else {
                        const _Float16* am = g.w.a + bt * g.w.mp * (size_t)g.w.ldm;
                        const h4 hi = *reinterpret_cast<const h4*>(am + across);
                        h4 lo{};
                        if (P == 3) lo = *reinterpret_cast<const h4*>(am + across + 32);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            v[e] = g.b * ((float)hi[e] + (float)lo[e]) + (g.c / kScaleA) * v[e];
                    }
                    h4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        _Float16 x, y;
                        split_hl(v[e], x, y);
                        hi[e] = x; lo[e] = y;
                    }
                    // a tile on the diagonal holds both halves itself, and stores one of them
                    if (ti != tj) {
                        *reinterpret_cast<h4*>(m + across) = hi;
                        if (P == 3) *reinterpret_cast<h4*>(m + across + 32) = lo;
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const size_t o = at<P>(i + e, g.w.ldm, j);
                        m[o] = hi[e];
                        if (P == 3) m[o + 32] = lo[e];
                    }
                } else {
                    const _Float16* y = g.w.y[g.cur] + bt * g.w.np * (size_t)g.w.ldm;
                    const size_t o = at<P>(j, g.w.ldm, i);
                    _Float16* ylo = P == 1 ? g.w.y_lo + (bt * g.w.np + j) * g.w.mp + i : nullptr;
                    const h4 xh = *reinterpret_cast<const h4*>(y + o);
                    const h4 xl = *reinterpret_cast<const h4*>(P == 3 ? y + o + 32 : ylo);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = g.a * ((float)xh[e] + (float)xl[e]) + v[e] * (1.0f / kScaleA);
                    if (MODE == kLast) {
                        const OutArgs& t = g.out;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int row = t.tall ? j : i + e, col = t.tall ? i + e : j;
                            if (row < t.rows && col < t.cols)
                                put_out(t, bt * t.stride + (size_t)row * t.ld + col, v[e] * (1.0f / kScaleX));
                        }
                    } else {
                        h4 hi, lo;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            _Float16 p, r;
                            split_hl(v[e], p, r);
                            hi[e] = p; lo[e] = r;
                        }
                        _Float16* yn = g.w.y[g.cur ^ 1] + bt * g.w.np * (size_t)g.w.ldm;
                        *reinterpret_cast<h4*>(yn + o) = hi;
                        *reinterpret_cast<h4*>(P == 3 ? yn + o + 32 : ylo) = lo;
                        _Float16* x = g.w.x + bt * g.w.mp * (size_t)g.w.ldn;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const size_t ox = at<P>(i + e, g.w.ldn, j);
                            x[ox] = hi[e];
                            if (P == 3) x[ox + 32] = lo[e];
                        }
                    }
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
        const float v = (float)y[o] + (float)(P == 3 ? y[o + 32] : w.y_lo[(bt * w.np + j) * w.mp + i]);
        put_out(t, bt * t.stride + (size_t)r * t.ld + c, v * (1.0f / kScaleX));
    }
}

// ---- plan ------------------------------------------------------------------------------
struct Plan {
    int tile, mp, np, ldm, ldn;
    size_t part, x, y, y_lo, ab, total;   // bytes
};
size_t round_up(size_t v, size_t q) { return (v + q - 1) / q * q; }
// Tiles of 128 where they fill the machine, of 64 where they would leave most of it idle.
Plan make_plan(int batch, int rows, int cols, int products) {
    Plan p{};
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    const int64_t big = (int64_t)((m + 127) / 128) * ((n + 127) / 128) * batch;
    p.tile = big >= 192 ? 128 : 64;
    p.mp = (int)round_up(m, p.tile);
    p.np = (int)round_up(n, p.tile);
    const int planes = products == 3 ? 2 : 1;
    p.ldm = p.mp * planes;
    p.ldn = p.np * planes;
    const size_t h = sizeof(_Float16);
    p.part = round_up((size_t)batch * kNormGroups * sizeof(double), 256);
    p.x = round_up((size_t)batch * p.mp * p.ldn * h, 256);
    p.y = round_up((size_t)batch * p.np * p.ldm * h, 256);
    p.y_lo = products == 1 ? round_up((size_t)batch * p.np * p.mp * h, 256) : 0;
    p.ab = round_up((size_t)batch * p.mp * p.ldm * h, 256);
    p.total = p.part + p.x + 2 * p.y + p.y_lo + 2 * p.ab;
    return p;
}

template <int P, int MODE, int WM, int WN, int FM, int FN>
void run_mul(MulArgs g, int batch, hipStream_t st) {
    constexpr int TM = 32 * WM * FM, TN = 32 * WN * FN;
    g.tiles_i = g.w.mp / TM;
    g.tiles_j = (MODE == kGram || MODE == kPoly ? g.w.mp : g.w.np) / TN;
    const int tiles = MODE == kGram || MODE == kPoly ? g.tiles_i * (g.tiles_i + 1) / 2 : g.tiles_i * g.tiles_j;
    hipLaunchKernelGGL((k_ortho_mul<P, MODE, WM, WN, FM, FN>), dim3(tiles, batch), dim3(64 * WM * WN), 0, st, g);
}
template <int P, int MODE>
void run_mul(const MulArgs& g, int tile, int batch, hipStream_t st) {
    if (tile == 128) run_mul<P, MODE, 2, 2, 2, 2>(g, batch, st);
    else run_mul<P, MODE, 2, 2, 1, 1>(g, batch, st);
}

template <int P>
int run_all(const InArgs& in, const OutArgs& out, int batch, int steps, const float* coef, const Plan& p, char* work,
            hipStream_t st) {
    Work w{};
    InArgs a = in;
    a.part = (double*)work;             work += p.part;
    w.x = (_Float16*)work;              work += p.x;
    w.y[0] = (_Float16*)work;           work += p.y;
    w.y[1] = (_Float16*)work;           work += p.y;
    w.y_lo = P == 1 ? (_Float16*)work : nullptr; work += p.y_lo;
    w.a = (_Float16*)work;              work += p.ab;
    w.b = (_Float16*)work;
    w.mp = p.mp; w.np = p.np; w.ldm = p.ldm; w.ldn = p.ldn;
    const int tall = out.tall;
    hipLaunchKernelGGL(k_ortho_norm, dim3(kNormGroups, batch), dim3(256), 0, st, a);
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
        g.l = g.r = w.x; g.ldl = g.ldr = p.ldn; g.l_batch = g.r_batch = xb; g.stages = p.ldn / 64;
        run_mul<P, kGram>(g, p.tile, batch, st);
        g.l = g.r = w.a; g.ldl = g.ldr = p.ldm; g.l_batch = g.r_batch = ab; g.stages = p.ldm / 64;
        run_mul<P, kPoly>(g, p.tile, batch, st);
        g.l = w.b; g.r = w.y[g.cur]; g.ldl = g.ldr = p.ldm; g.l_batch = ab; g.r_batch = yb; g.stages = p.ldm / 64;
        if (s + 1 < steps) run_mul<P, kStep>(g, p.tile, batch, st);
        else run_mul<P, kLast>(g, p.tile, batch, st);
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
    const int p = products ? products : dtype == CFP_BF16 ? 1 : 3;
    const Plan plan = make_plan(batch, rows, cols, p);
    CFP_REQUIRE(d_work && work_bytes >= plan.total && (reinterpret_cast<uintptr_t>(d_work) & 255u) == 0,
                "cfp_orthogonalize: needs a 256-byte aligned workspace of %zu bytes (got %zu)", plan.total, work_bytes);
    float c[3 * kMaxSteps];
    fill_coef(coefs, steps, c);
    InArgs in{};
    in.g = d_g; in.dtype = dtype; in.ld = ld; in.stride = batch_stride; in.rows = rows; in.cols = cols; in.eps = eps;
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
    CFP_REQUIRE(u.work && u.work_bytes >= plan.total && (reinterpret_cast<uintptr_t>(u.work) & 255u) == 0,
                "cfp_muon_update: needs a 256-byte aligned workspace of %zu bytes (got %zu)", plan.total, u.work_bytes);
    float c[3 * kMaxSteps];
    fill_coef(u.coefs, u.steps, c);
    InArgs in{};
    in.g = u.g; in.dtype = CFP_F32; in.ld = u.ld; in.stride = u.stride; in.rows = u.rows; in.cols = u.cols;
    in.mom = u.mom; in.beta = u.beta; in.nesterov = u.nesterov; in.eps = u.eps;
    in.g_clear = u.clear_g ? u.g : nullptr;
    OutArgs out{};
    out.out = u.w; out.dtype = CFP_F32; out.ld = u.ld; out.stride = u.stride;
    out.rows = u.rows; out.cols = u.cols; out.tall = u.rows > u.cols;
    out.update = 1; out.lr_dev = u.lr_dev; out.lr = u.lr; out.decay = u.decay;
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
