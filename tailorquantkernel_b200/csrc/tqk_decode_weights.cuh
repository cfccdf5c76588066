// tqk_decode_weights.cuh -- the weight pass of tqk_decode_q8_weights (included
// by tqk_decode.cu): turns the scores and the final (max, sum) of every q head,
// which the decode kernels leave behind with WT != WT_NONE, into each cached
// row's attention weight summed over the q heads of its kv head, and adds it to
// the row's running sum.
#pragma once

namespace tqk {

constexpr int WP_THREADS = 128;
constexpr int WP_TOKENS = 4;   // tokens per thread, WP_THREADS apart: every load and store is coalesced
constexpr int WP_HEADS = 4;    // q heads whose scores are in flight together: 16 loads per thread

// weight_out[t] = weight[t] + sum_g e^{s_g[t] - m_g} / l_g, g over the kv head's q heads in order.  Bound
// by L2 and DRAM: 4 * group bytes of scores, which the decode has just written, and 8 bytes of sums per
// cached row, against the 2 * (head_dim / 32) * 36 bytes of K and V that the decode streams.
template <int WT>
__global__ void __launch_bounds__(WP_THREADS) weight_sum_kernel(const DecodeParams p) {
    const int item = blockIdx.z, kvh = blockIdx.y;
    const int t0 = blockIdx.x * (WP_THREADS * WP_TOKENS) + threadIdx.x;
    const long long at = (long long)item * p.stat_stride + (long long)kvh * p.max_tokens;
    grid_dependency_wait();
    grid_dependents_launch();
    int len = p.lens ? p.lens[item] : p.len0 + item * p.len_step;
    len = min(max(len, 0), p.len_cap);  // as the decode clamped (and reported) it
    if (t0 - (int)threadIdx.x >= len) return;

    const long long head0 = (long long)item * (p.n_kv * p.group) + kvh * p.group;
    const float *src = p.scores + head0 * p.score_stride;
    int from[WP_TOKENS];  // tokens behind the end load the last one's scores
#pragma unroll
    for (int k = 0; k < WP_TOKENS; k++) from[k] = min(t0 + k * WP_THREADS, len - 1);
    // the sums, usually written by the pass before, are in flight together with the first scores
    float old[WP_TOKENS];
#pragma unroll
    for (int k = 0; k < WP_TOKENS; k++) old[k] = p.weight[at + from[k]];
    float w[WP_TOKENS] = {};
    bool whole = true;
    for (int g0 = 0; g0 < p.group; g0 += WP_HEADS) {
        float s[WP_HEADS][WP_TOKENS];
        float2 ml[WP_HEADS];
#pragma unroll
        for (int g = 0; g < WP_HEADS; g++) {
            const int h = min(g0 + g, p.group - 1);
            ml[g] = p.ml[head0 + h];
#pragma unroll
            for (int k = 0; k < WP_TOKENS; k++) s[g][k] = src[h * p.score_stride + from[k]];
        }
#pragma unroll
        for (int g = 0; g < WP_HEADS; g++) {
            if (g0 + g >= p.group) break;
            whole &= !is_unfinished(ml[g]);
            const float inv = __fdiv_rn(1.0f, ml[g].y);
#pragma unroll
            for (int k = 0; k < WP_TOKENS; k++) {
                const float d = s[g][k] - ml[g].x;
                w[k] = fmaf(WT == WT_LOG2 ? ex2f(d) : expf(d), inv, w[k]);
            }
        }
    }
    if (!whole) return;  // the decode gave up on a wait (and recorded it)
#pragma unroll
    for (int k = 0; k < WP_TOKENS; k++) {
        const int t = t0 + k * WP_THREADS;
        if (t >= len) continue;
        const bool fresh = p.k_new && t == len - 1;
        p.weight_out[at + t] = fresh ? w[k] : old[k] + w[k];
        if (fresh && p.position) p.position[at + t] = p.new_pos ? p.new_pos[item] : p.new_pos0;
    }
}

}  // namespace tqk
