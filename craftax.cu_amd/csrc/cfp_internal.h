// Library-internal definition of the policy object (opaque in include/cfp.h).
#pragma once

#include <numeric>

#include "cfp_common.h"

struct cfp_policy {
    int n = 0;
    int layers = 0;
    int variant = 0;   // 0 full game, 1 classic
    size_t param_count = 0;
    float* params = nullptr;
    float* we_pk = nullptr;
    uint16_t* we_s3 = nullptr;    // map rows of W_enc split in three bf16 terms
    float* wg_pk = nullptr;
    float* wav_pk = nullptr;
    uint16_t* we_bf = nullptr;    // bf16 mirrors (MFMA 32x32x16 order)
    uint16_t* wg_bf = nullptr;
    uint16_t* wav_bf = nullptr;
    int gemm_bf16 = 0;            // forward entry points run the bf16-input kernel
    int rs_bf16 = 0;              // r_state rows leave as bf16 (a trainer with a bf16 state slab)
    void* enc_x9 = nullptr;       // split mirror of W_enc for the forward from a feature matrix
    void* t16 = nullptr;          // mirrors of the 16-env-tile kernel (full game only)
    int small_tiles = 0;          // batches of at most 4096 envs run on 16-env tiles
    float* h_state = nullptr;
    uint8_t* rec = nullptr;
    float* h_enc = nullptr;
    float* h3 = nullptr;
    float* logits = nullptr;
    hipStream_t stream = nullptr;
};

namespace cfp {
// weight pointers, variant and action count of a policy into launch arguments
void fill_forward_weights(const cfp_policy* p, FwdArgs& a);

// Sampler behind cfp_value_sample.  From kSampleRowsFrom envs on it runs one thread per
// env; below, sixteen lanes per env, and there `ticket` (one zeroed word of device
// memory, or null) makes the launch bump *d_step_ctr itself once every workgroup has
// read it.
constexpr int kSampleRowsFrom = 16384;
int value_sample(const float* d_av, int n, int actions, float* d_env_actions, int32_t* d_actions,
                 float* d_logprobs, float* d_values, uint64_t seed, const uint64_t* d_step_ctr,
                 unsigned* ticket, hipStream_t st);

// launch_forward also draws the actions (FwdArgs::s_act ...) when this holds: full-game
// records in recording mode on 32-env tiles, one tile per workgroup (at most one per CU).
bool forward_draws(const FwdArgs& a);

// Whether two batches of `batch` matrices rows x cols (elements of `bytes`, row strides ld, matrix
// strides `stride`) share no entry, where that shows: address ranges apart, or whole matrices or
// columns side by side in a period that all strides are multiples of.
inline bool apart(const void* a, int64_t ld_a, int64_t stride_a, const void* b, int64_t ld_b, int64_t stride_b, int batch, int rows,
                  int cols, size_t bytes) {
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    const int64_t span_a = (int64_t)(rows - 1) * ld_a + cols, span_b = (int64_t)(rows - 1) * ld_b + cols;
    const uintptr_t a1 = a0 + ((batch - 1) * stride_a + span_a) * bytes, b1 = b0 + ((batch - 1) * stride_b + span_b) * bytes;
    if (a1 <= b0 || b1 <= a0) return true;
    const int64_t d = (int64_t)(b0 - a0) / (int64_t)bytes;
    auto beside = [d](int64_t period, int64_t len_a, int64_t len_b) {
        if (period <= 0) return false;
        const int64_t from = (d % period + period) % period;
        return from >= len_a && from <= period - len_b;
    };
    const int64_t matrices = batch > 1 ? std::gcd(stride_a, stride_b) : 0, lines = rows > 1 ? std::gcd(ld_a, ld_b) : 0;
    return beside(matrices, span_a, span_b) || beside(std::gcd(matrices, lines), cols, cols);
}

// One Muon step of a batch of fp32 matrices that share ld and stride (orthogonalize.hip,
// cfp_muon_update); clear_g: the gradient is zeroed behind its last read.
struct MuonArgs {
    float* w;
    float* g;
    float* mom;
    int64_t ld, stride;
    int batch, rows, cols;
    const float* lr_dev;   // or null: factor of lr in device memory
    float lr, beta;
    int nesterov;
    float decay, scale;    // scale 0: sqrt(max(1, rows / cols))
    int steps;
    const float* coefs;    // host [steps][3] or null
    float eps;
    int products;          // 0 (= 3), 1 or 3
    void* work;
    size_t work_bytes;
    int clear_g;
};
int muon_update(const MuonArgs& u, hipStream_t st);

// One rollout step's policy side for the trainer: records -> heads into the policy's
// live state and logits (r_state recorded), then the draw into act / logp / value
// (and env_actions when not null) with offset *step_ctr, then *step_ctr += 1.  One
// launch where the 16-env-tile kernel applies, forward + sampler otherwise.
struct SampleOut {
    int32_t* act;
    float* logp;
    float* value;
    float* env_actions;
    uint64_t seed;
    uint64_t* step_ctr;
    unsigned* ticket;   // one zeroed word, left zeroed
};
int forward_and_sample(cfp_policy* p, const uint8_t* d_rec_row, const float* d_terminals,
                       float* d_r_state_t, int n, const SampleOut& s, hipStream_t st);
}  // namespace cfp
