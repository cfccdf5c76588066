// tqk_logits.cu -- constraints on the next token (tqk_process_logits):
// repetition, frequency and presence penalties over each row's history, token
// biases, a grammar's bit mask, and the greedy choice among what is left.
//
// One thread-block cluster per row, a contiguous part of the vocabulary per CTA,
// worked through in pieces of LG_PIECE tokens: the piece's logits are loaded into
// registers first (8 16-byte loads in flight per thread); while they are on
// their way, the row's history is scanned and the piece's tokens are counted in
// shared memory (a word per token: bit 31 seen, bit 30 in the bias list, the rest
// the count after the prompt; integer atomics, so the order does not show); then
// penalties, biases and mask are applied in registers and the piece is stored
// once.  Every logit is read and written once: 8 bytes of DRAM traffic per token
// bound the kernel, and the history costs 4 bytes per entry and CTA, from L2.
// The CTAs' largest values meet through distributed shared memory.
#include "tqk_internal.h"

#include <mutex>

namespace tqk {
namespace {

constexpr int LG_THREADS = 512;
constexpr int LG_PER_THREAD = 32;                        // logits per thread and piece, in registers
constexpr int LG_PIECE = LG_THREADS * LG_PER_THREAD;     // 16384 tokens
constexpr int LG_CLUSTER = 8;                            // most CTAs per row (portable cluster size)
constexpr uint32_t LG_SEEN = 0x80000000u, LG_BIASED = 0x40000000u, LG_COUNT = 0x3FFFFFFFu;

struct LogitsParams {
    const float *logits;
    long long logits_stride;
    float *out;
    long long out_stride;
    int *choice;
    int n_rows, vocab;
    const int *tokens, *token_offsets;
    int n_tokens;
    const int *prompt_lens;
    const float *repetition, *frequency, *presence;
    const int *bias_tokens;
    const float *bias_values;
    const int *bias_offsets;
    int n_bias;
    const uint32_t *mask;
    long long mask_stride;
    const int *mask_rows;
    int n_mask_rows;
    int per_cta;  // tokens per CTA, a multiple of 128
    int *err;
};

// Entries [b, e) of row r in a packed list of n, clamped.
__device__ __forceinline__ void list_range(const int *offsets, int r, int n, int *err, bool report, int &b, int &e) {
    const int b0 = offsets[r], e0 = offsets[r + 1];
    b = min(max(b0, 0), n);
    e = min(max(e0, b), n);
    if (report && (b != b0 || e != e0)) record_error(err, DEVERR_BADLEN);
}

// A candidate for the greedy choice: the largest value, the first token of it (token < 0: none yet).
struct Best {
    float v;
    int token;
};
__device__ __forceinline__ Best better(Best a, Best b) {
    const bool take = b.token >= 0 && (a.token < 0 || b.v > a.v || (b.v == a.v && b.token < a.token));
    return take ? b : a;
}

// VEC: rows are 16-byte aligned (4 consecutive tokens per load); else one token per load, the warp's consecutive.
// COUNT: the call has histories or biases.
template <bool VEC, bool COUNT>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitsParams p) {
    extern __shared__ __align__(16) uint32_t counts[];  // [piece], with COUNT
    __shared__ Best warp_best[LG_THREADS / 32];
    __shared__ Best cta_best;
    grid_dependency_wait();
    grid_dependents_launch();
    constexpr int W = VEC ? 4 : 1;                 // tokens per load
    constexpr int STEP = LG_THREADS * W;           // tokens between a thread's loads
    constexpr int LOADS = LG_PER_THREAD / W;
    const int tid = threadIdx.x, C = (int)gridDim.x, rank = (int)blockIdx.x, row = blockIdx.y;
    const float *src = p.logits + (long long)row * p.logits_stride;
    float *dst = p.out ? p.out + (long long)row * p.out_stride : nullptr;
    const int v0 = min(p.vocab, rank * p.per_cta), v1 = min(p.vocab, v0 + p.per_cta);
    const bool report = rank == 0 && tid == 0;

    int h0 = 0, h1 = 0, prompt_end = 0, b0 = 0, b1 = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if constexpr (COUNT) {
        if (p.tokens) {
            list_range(p.token_offsets, row, p.n_tokens, p.err, report, h0, h1);
            const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
            prompt_end = h0 + min(max(prompt, 0), h1 - h0);
            if (p.repetition) rep = p.repetition[row];
            if (p.frequency) freq = p.frequency[row];
            if (p.presence) pres = p.presence[row];
        }
        if (p.bias_tokens) list_range(p.bias_offsets, row, p.n_bias, p.err, report, b0, b1);
    }
    const uint32_t *mask = nullptr;
    bool barred = false;  // a bad mask row index allows nothing
    if (p.mask) {
        const int m = p.mask_rows ? p.mask_rows[row] : row;
        barred = m < -1 || m >= p.n_mask_rows;
        if (barred && report) record_error(p.err, DEVERR_BADLEN);
        if (m >= 0 && !barred) mask = p.mask + (long long)m * p.mask_stride;
    }

    Best best{-INFINITY, -1};
    for (int t0 = v0; t0 < v1; t0 += LG_PIECE) {
        const int n = min(LG_PIECE, v1 - t0);
        float x[LOADS][W];
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
            const int i = tid * W + k * STEP;
            if constexpr (VEC) {
                if (i + W <= n) {
                    const float4 f = *reinterpret_cast<const float4 *>(src + t0 + i);
                    x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
                } else {
#pragma unroll
                    for (int j = 0; j < W; j++) x[k][j] = i + j < n ? src[t0 + i + j] : 0.0f;
                }
            } else {
                x[k][0] = i < n ? src[t0 + i] : 0.0f;
            }
        }
        if constexpr (COUNT) {
            for (int i = tid * 4; i < n; i += LG_THREADS * 4) *reinterpret_cast<uint4 *>(counts + i) = uint4{0, 0, 0, 0};
            __syncthreads();
            for (int i = h0 + tid; i < h1; i += LG_THREADS) {
                const unsigned t = (unsigned)p.tokens[i] - (unsigned)t0;
                if (t >= (unsigned)n) continue;
                if (i < prompt_end) atomicOr(&counts[t], LG_SEEN);
                else atomicAdd(&counts[t], 1u);
            }
            for (int i = b0 + tid; i < b1; i += LG_THREADS) {
                const unsigned t = (unsigned)p.bias_tokens[i] - (unsigned)t0;
                if (t < (unsigned)n) atomicOr(&counts[t], LG_BIASED);
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
            const int i = tid * W + k * STEP;
            if (i >= n) break;
            const uint32_t allowed = barred ? 0u : mask ? mask[(t0 + i) >> 5] >> ((t0 + i) & 31) : 0xFFFFFFFFu;
            uint32_t c[W] = {};
            if constexpr (COUNT) {
                if constexpr (VEC) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(counts + i);
                    c[0] = u.x; c[1] = u.y; c[2] = u.z; c[3] = u.w;
                } else {
                    c[0] = counts[i];
                }
            }
#pragma unroll
            for (int j = 0; j < W; j++) {
                float v = x[k][j];
                if (COUNT && c[j]) {
                    const uint32_t made = c[j] & LG_COUNT;
                    if (p.repetition && (c[j] & (LG_SEEN | LG_COUNT))) v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (made) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, __uint2float_rn(made))), pres);
                    if (c[j] & LG_BIASED) {
                        float s = 0.0f;
                        for (int q = b0; q < b1; q++)
                            if (p.bias_tokens[q] == t0 + i + j) s = __fadd_rn(s, p.bias_values[q]);
                        v = __fadd_rn(v, s);
                    }
                }
                if (!((allowed >> j) & 1u)) v = -INFINITY;
                if (i + j < n && v > best.v) best = Best{v, t0 + i + j};
                x[k][j] = v;
            }
            if (dst) {
                if constexpr (VEC) {
                    if (i + W <= n) {
                        *reinterpret_cast<float4 *>(dst + t0 + i) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < W; j++)
                            if (i + j < n) dst[t0 + i + j] = x[k][j];
                    }
                } else {
                    dst[t0 + i] = x[k][0];
                }
            }
        }
        if (COUNT && t0 + LG_PIECE < v1) __syncthreads();  // the next piece clears the counts
    }

    // ---- the greedy choice (the same branch for every CTA of the cluster)
    if (!p.choice) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = tid < LG_THREADS / 32 ? warp_best[tid] : Best{-INFINITY, -1};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
        if (tid == 0) cta_best = best;
    }
    if (C == 1) {
        if (tid == 0) p.choice[row] = best.token;
        return;
    }
    __syncwarp();
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
        for (int r = 1; r < C; r++) {
            const uint32_t a = cluster_map(&cta_best, (uint32_t)r);
            best = better(best, Best{ld_cluster_f32(a), (int)ld_cluster_u32(a + 4)});
        }
        p.choice[row] = best.token;
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while its candidate is read
}

template <bool VEC, bool COUNT>
int launch_logits(const LogitsParams &p, int cluster, cudaStream_t stream) {
    const int piece = p.per_cta < LG_PIECE ? p.per_cta : LG_PIECE;
    const size_t smem = COUNT ? (size_t)piece * sizeof(uint32_t) : 0;
    if (COUNT) {
        // the dynamic shared-memory opt-in is a per-device function attribute
        static std::mutex mu;
        static bool ready[64];
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || dev < 0 || dev >= 64) return fail_cuda(e, "tqk_process_logits: cudaGetDevice");
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(logits_kernel<VEC, COUNT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     LG_PIECE * (int)sizeof(uint32_t));
            if (e != cudaSuccess) return fail_cuda(e, "tqk_process_logits: kernel attributes");
            ready[dev] = true;
        }
    }
    const dim3 grid((unsigned)cluster, (unsigned)p.n_rows);
    if (cluster == 1) return launch_pdl(logits_kernel<VEC, COUNT>, grid, dim3(LG_THREADS), smem, stream, p);
    return launch_pdl_cluster(logits_kernel<VEC, COUNT>, grid, dim3(LG_THREADS), smem, stream, (unsigned)cluster, p);
}

}  // namespace
}  // namespace tqk

using namespace tqk;

extern "C" int tqk_process_logits(const tqk_logits_args *a, tqk_stream_t stream) {
    if (!a) return fail(TQK_EINVAL, "tqk_process_logits: NULL args");
    if (a->n_rows <= 0 || a->vocab_size <= 0) return fail(TQK_EINVAL, "tqk_process_logits: non-positive shape");
    // token indexes and counts are 30 bits (a word per token also carries two flags)
    if (a->vocab_size > (int)LG_COUNT || a->n_tokens > (int)LG_COUNT)
        return fail(TQK_EUNSUPPORTED, "tqk_process_logits: vocab_size or n_tokens above 2^30 - 1");
    if (a->n_rows > 65535) return fail(TQK_EINVAL, "tqk_process_logits: n_rows > 65535");
    if (!a->logits || (!a->out && !a->choice))
        return fail(TQK_EINVAL, "tqk_process_logits: NULL logits, or neither out nor choice");
    const int64_t ls = a->logits_stride ? a->logits_stride : a->vocab_size;
    const int64_t os = a->out_stride ? a->out_stride : a->vocab_size;
    const int64_t words = ((int64_t)a->vocab_size + 31) / 32, ms = a->mask_stride ? a->mask_stride : words;
    if (a->n_rows > 1 && (ls < a->vocab_size || os < a->vocab_size))
        return fail(TQK_EINVAL, "tqk_process_logits: a row stride below vocab_size");
    if (a->out == a->logits && a->n_rows > 1 && ls != os)
        return fail(TQK_EINVAL, "tqk_process_logits: in place, out_stride must be logits_stride");
    if (a->tokens ? !a->token_offsets || a->n_tokens < 0 : a->repetition || a->frequency || a->presence || a->prompt_lens)
        return fail(TQK_EINVAL, "tqk_process_logits: penalties need tokens and token_offsets");
    if (a->bias_tokens ? !a->bias_values || !a->bias_offsets || a->n_bias < 0 : a->bias_values != nullptr)
        return fail(TQK_EINVAL, "tqk_process_logits: bias_tokens, bias_values and bias_offsets go together");
    if (a->mask && (ms < words || a->n_mask_rows < (a->mask_rows ? 0 : a->n_rows)))
        return fail(TQK_EINVAL, "tqk_process_logits: mask_stride or n_mask_rows too small");
    if (!a->mask && a->mask_rows) return fail(TQK_EINVAL, "tqk_process_logits: mask_rows without mask");
    const void *arrays[] = {a->logits, a->out, a->choice, a->tokens, a->token_offsets, a->prompt_lens, a->repetition,
                            a->frequency, a->presence, a->bias_tokens, a->bias_values, a->bias_offsets, a->mask,
                            a->mask_rows};
    for (const void *q : arrays)
        if (reinterpret_cast<uintptr_t>(q) & 3) return fail(TQK_EALIGN, "tqk_process_logits: arrays must be 4-byte aligned");
    int rc = ensure_device();
    if (rc) return rc;
    LogitsParams p{};
    p.logits = a->logits;
    p.logits_stride = ls;
    p.out = a->out;
    p.out_stride = os;
    p.choice = a->choice;
    p.n_rows = a->n_rows;
    p.vocab = a->vocab_size;
    const bool penal = a->tokens && (a->repetition || a->frequency || a->presence);
    if (penal) {
        p.tokens = a->tokens;
        p.token_offsets = a->token_offsets;
        p.n_tokens = a->n_tokens;
        p.prompt_lens = a->prompt_lens;
        p.repetition = a->repetition;
        p.frequency = a->frequency;
        p.presence = a->presence;
    }
    p.bias_tokens = a->bias_tokens;
    p.bias_values = a->bias_values;
    p.bias_offsets = a->bias_offsets;
    p.n_bias = a->n_bias;
    p.mask = a->mask;
    p.mask_stride = ms;
    p.mask_rows = a->mask_rows;
    p.n_mask_rows = a->n_mask_rows;
    p.err = device_info()->err_word;
    // CTAs per row: as many as the portable cluster has while each keeps a few thousand tokens
    int cluster = (a->vocab_size + 2047) / 2048;
    if (cluster > LG_CLUSTER) cluster = LG_CLUSTER;
    p.per_cta = (int)((((int64_t)a->vocab_size + cluster - 1) / cluster + 127) / 128 * 128);
    const bool vec = ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 &&
                     (a->n_rows == 1 || ((ls | (p.out ? os : 0)) & 3) == 0);
    const bool count = penal || a->bias_tokens;
    cudaStream_t st = (cudaStream_t)stream;
    if (vec) return count ? launch_logits<true, true>(p, cluster, st) : launch_logits<true, false>(p, cluster, st);
    return count ? launch_logits<false, true>(p, cluster, st) : launch_logits<false, false>(p, cluster, st);
}
