// tqk_decode_weights.cuh -- the weight pass of tqk_decode_q8_weights (included
// by tqk_decode.cu): turns the scores and the final (max, sum) of every q head,
// which the decode kernels leave behind with WT != WT_NONE, into each cached
// row's attention weight summed over the q heads of its kv head, and adds it to
// the row's running sum.
#pragma once

namespace tqk {

constexpr int WP_THREADS = 256;
constexpr int WP_TOKENS = 4;   // tokens per thread, WP_THREADS apart: every load and store is coalesced
constexpr int WP_HEADS = 256;  // q heads whose (max, 1 / sum) fit in shared memory at a time

struct WeightParams {
    const float *scores;  // [item][q head][score_stride]
    long long score_stride;
    const float2 *ml;     // [item][q head] final {max, sum}
    int group, n_kv, max_tokens, len_cap;
    const int *lens;
    int len0, len_step;
    const float *weight;
    float *weight_out;
    long long item_stride;  // elements between items' sums (and positions)
    int appended;           // slot len - 1 holds a row of this call: its sum starts from 0
    int *position;
    const int *new_pos;
    int new_pos0;
};

// weight_out[t] = weight[t] + sum_g e^{s_g[t] - m_g} / l_g, g over the kv head's q heads in order.  Bound
// by L2 and DRAM: 4 * group bytes of scores, which the decode has just written, and 8 bytes of sums per
// cached row, against the 2 * (head_dim / 32) * 36 bytes of K and V that the decode streams.
template <int WT>
__global__ void __launch_bounds__(WP_THREADS) weight_sum_kernel(const WeightParams p) {
    grid_dependency_wait();
    grid_dependents_launch();
    const int item = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x;
    int len = p.lens ? p.lens[item] : p.len0 + item * p.len_step;
    len = min(max(len, 0), p.len_cap);  // as the decode clamped (and reported) it
    const int t0 = blockIdx.x * (WP_THREADS * WP_TOKENS);
    if (t0 >= len) return;

    __shared__ float2 ml[WP_HEADS];
    const long long head0 = (long long)item * (p.n_kv * p.group) + kvh * p.group;
    float w[WP_TOKENS] = {};
    for (int g0 = 0; g0 < p.group; g0 += WP_HEADS) {
        const int n = min(WP_HEADS, p.group - g0);
        if (g0) __syncthreads();
        for (int g = tid; g < n; g += WP_THREADS) {
            const float2 v = p.ml[head0 + g0 + g];
            ml[g] = make_float2(v.x, __fdiv_rn(1.0f, v.y));
        }
        __syncthreads();
        const float *src = p.scores + (head0 + g0) * p.score_stride + t0 + tid;
        for (int g = 0; g < n; g++, src += p.score_stride) {
            const float2 v = ml[g];
#pragma unroll
            for (int k = 0; k < WP_TOKENS; k++) {
                if (t0 + tid + k * WP_THREADS >= len) continue;
                const float d = src[k * WP_THREADS] - v.x;
                w[k] = fmaf(WT == WT_LOG2 ? ex2f(d) : expf(d), v.y, w[k]);
            }
        }
    }

    const long long at = (long long)item * p.item_stride + (long long)kvh * p.max_tokens;
#pragma unroll
    for (int k = 0; k < WP_TOKENS; k++) {
        const int t = t0 + tid + k * WP_THREADS;
        if (t >= len) continue;
        const bool fresh = p.appended && t == len - 1;
        p.weight_out[at + t] = fresh ? w[k] : p.weight[at + t] + w[k];
        if (fresh && p.position) p.position[at + t] = p.new_pos ? p.new_pos[item] : p.new_pos0;
    }
}

}  // namespace tqk
