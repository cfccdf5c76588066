// tqk_logits.cu -- constraints on the next token (tqk_process_logits):
// repetition, frequency and presence penalties over each row's history, token
// biases, a grammar's bit mask, and the greedy choice among what is left.
//
// One thread-block cluster per row; blocks of 128 tokens are dealt out to its
// CTAs in turn.  The bulk of a row -- tokens in neither its history nor its bias
// list -- only meets the mask and is streamed through registers: 8 16-byte loads
// in flight per thread, each logit read and written once, which is the kernel's
// floor (8 bytes of DRAM traffic per token).  Around the stream:
//   * while the first logits are on their way, every CTA scans the history and
//     counts its own tokens in shared memory (a counter per token: seen, in the
//     bias list, and the count after the prompt; integer atomics, so their order
//     does not show).  Frequent tokens have neighbouring ids in many vocabularies;
//     dealing out small blocks spreads them over the CTAs;
//   * the stream leaves counted tokens alone and puts them on a list; the list is
//     worked off with full warps, so the division and the branches of the
//     penalties cost by the distinct tokens of the history, not by the vocabulary;
//     the next logits are loaded meanwhile;
//   * each CTA pushes its candidate for the greedy choice to the first CTA's
//     shared memory and leaves.
#include "tqk_internal.h"

#include <climits>
#include <mutex>

namespace tqk {
namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_WARPS = LG_THREADS / 32;
constexpr int LG_BLOCK = 128;                            // tokens per block: a warp's 16-byte loads
constexpr int LG_LOADS = 8;                              // blocks per warp and chunk, in registers
constexpr int LG_CHUNK = LG_WARPS * LG_LOADS * LG_BLOCK; // 8192 tokens
constexpr int LG_CLUSTER = 16;                           // most CTAs per row (non-portable above 8), a power of two
constexpr int LG_COUNT_BYTES_MAX = 64 << 10;             // counters per CTA
constexpr int LG_SCAN = 8;                               // history entries in flight per thread

// Counters: 16 bits per token (two to a word) for histories of up to LG_SHORT entries, else 32 bits.  From the top:
// seen, in the bias list, more than once in the bias list, and the count after the prompt.
constexpr int LG_SHORT = (1 << 13) - 1;
template <bool SHORT>
struct Counter {
    static constexpr int BITS = SHORT ? 16 : 32;
    static constexpr uint32_t SEEN = 1u << (BITS - 1), BIASED = 1u << (BITS - 2), AGAIN = 1u << (BITS - 3);
    static constexpr uint32_t COUNT = AGAIN - 1;
    // the word of token t, and the place of its counter in it
    static __device__ __forceinline__ int word(int t) { return SHORT ? t >> 1 : t; }
    static __device__ __forceinline__ int shift(int t) { return SHORT ? (t & 1) * 16 : 0; }
    static __device__ __forceinline__ uint32_t get(const uint32_t *c, int t) {
        return SHORT ? (c[t >> 1] >> shift(t)) & 0xFFFFu : c[t];
    }
};
constexpr int LG_COUNT_MAX = Counter<false>::COUNT;

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
    int log_c;        // log2 of the CTAs per row
    int own_blocks;   // blocks per CTA
    int count_bytes;  // counters' shared memory, whole chunks
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

// What all threads of a CTA know of their row.
struct Row {
    const float *src;
    float *dst;
    const uint32_t *mask;  // or nullptr
    bool barred;           // a bad mask row index: nothing is allowed
    int h0, h1, prompt_end, b0, b1;
};

// Bit t of the row's mask.
__device__ __forceinline__ bool allowed_token(const Row &r, int t) {
    return !r.barred && (!r.mask || (r.mask[t >> 5] >> (t & 31)) & 1u);
}

// A listed token's final value: penalties by its counter c, then its biases' sum s.
template <bool SHORT>
__device__ __forceinline__ float constrained(const LogitsParams &p, const Row &r, int row, int t, uint32_t c, float s) {
    using K = Counter<SHORT>;
    float v = r.src[t];  // in place: still the logit
    if (p.repetition && (c & (K::SEEN | K::COUNT))) {
        const float rep = p.repetition[row];
        v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    }
    if (c & K::COUNT) {
        const float freq = p.frequency ? p.frequency[row] : 0.0f, pres = p.presence ? p.presence[row] : 0.0f;
        v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, __uint2float_rn(c & K::COUNT))), pres);
    }
    if (c & K::BIASED) v = __fadd_rn(v, s);
    return allowed_token(r, t) ? v : -INFINITY;
}

// The CTA's tokens: block b of the row is block b >> log_c of CTA b mod C.  The row's token at place i of them:
__device__ __forceinline__ int token_at(const LogitsParams &p, int i) {
    return (((i / LG_BLOCK) << p.log_c) + (int)blockIdx.x) * LG_BLOCK + i % LG_BLOCK;
}
// ... and the place of token `tok`, or -1 when it is another CTA's or outside the vocabulary.
__device__ __forceinline__ int place_of(const LogitsParams &p, int tok) {
    const int blk = tok / LG_BLOCK;
    if ((unsigned)tok >= (unsigned)p.vocab || (blk & ((1 << p.log_c) - 1)) != (int)blockIdx.x) return -1;
    return (blk >> p.log_c) * LG_BLOCK + tok % LG_BLOCK;
}

// The logits of the chunk at place t0, 8 blocks per warp.  VEC: tokens 4 lane .. 4 lane + 3 of each block; else tokens
// lane, 32 + lane, 64 + lane, 96 + lane.
template <bool VEC>
__device__ __forceinline__ void load_chunk(const LogitsParams &p, const float *src, int t0, float (&x)[LG_LOADS][4]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < LG_LOADS; k++) {
        const int first = token_at(p, t0 + (warp + k * LG_WARPS) * LG_BLOCK);
        if constexpr (VEC) {
            const int t = first + 4 * lane;
            if (t + 4 <= p.vocab) {
                const float4 f = *reinterpret_cast<const float4 *>(src + t);
                x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) x[k][j] = t + j < p.vocab ? src[t + j] : 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) x[k][j] = first + 32 * j + lane < p.vocab ? src[first + 32 * j + lane] : 0.0f;
        }
    }
}
// The warp's 32 mask words of the chunk, lane l holding word l % 4 of block l / 4.
__device__ __forceinline__ uint32_t load_words(const LogitsParams &p, const Row &r, int t0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t words = r.barred ? 0u : 0xFFFFFFFFu;
    if (r.mask) {
        const int t = token_at(p, t0 + (warp + (lane >> 2) * LG_WARPS) * LG_BLOCK) + 32 * (lane & 3);
        if (t < p.vocab) words = r.mask[t >> 5];
    }
    return words;
}

// This CTA's share of a row.  On entry x holds the first chunk, and the counters, which cover `span` tokens (whole
// chunks) at a time, and both list lengths are zero.
template <bool VEC, bool COUNT, bool SHORT>
__device__ __forceinline__ Best work_row(const LogitsParams &p, const Row &r, int row, int span, uint32_t *counts,
                                         uint16_t *list, int *n_listed, float (&x)[LG_LOADS][4]) {
    using K = Counter<SHORT>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int own = p.own_blocks * LG_BLOCK;
    Best best{-INFINITY, -1};
    uint32_t words = load_words(p, r, 0);
    for (int t0 = 0, c0 = 0, chunk = 0; t0 < own; t0 += LG_CHUNK, chunk++) {
        if constexpr (COUNT) {
            if (t0 == 0 || t0 == c0 + span) {
                // ---- the counters of the tokens from t0 on
                if (t0 > 0) {  // the last span's are done with (the barrier after its last list)
                    for (int i = tid; i < p.count_bytes / 16; i += LG_THREADS)
                        reinterpret_cast<uint4 *>(counts)[i] = uint4{0, 0, 0, 0};
                }
                c0 = t0;
                __syncthreads();
                for (int i0 = r.h0 + tid; i0 < r.h1; i0 += LG_SCAN * LG_THREADS) {
                    int tok[LG_SCAN];
#pragma unroll
                    for (int q = 0; q < LG_SCAN; q++) {
                        const int i = i0 + q * LG_THREADS;
                        tok[q] = i < r.h1 ? p.tokens[i] : -1;
                    }
#pragma unroll
                    for (int q = 0; q < LG_SCAN; q++) {
                        const int t = place_of(p, tok[q]) - c0;
                        if ((unsigned)t >= (unsigned)span) continue;
                        if (i0 + q * LG_THREADS < r.prompt_end) atomicOr(&counts[K::word(t)], K::SEEN << K::shift(t));
                        else atomicAdd(&counts[K::word(t)], 1u << K::shift(t));
                    }
                }
                for (int i = r.b0 + tid; i < r.b1; i += LG_THREADS) {
                    const int t = place_of(p, p.bias_tokens[i]) - c0;
                    if ((unsigned)t >= (unsigned)span) continue;
                    const uint32_t flag = K::BIASED << K::shift(t);
                    if (atomicOr(&counts[K::word(t)], flag) & flag) atomicOr(&counts[K::word(t)], K::AGAIN << K::shift(t));
                }
                __syncthreads();
            }
        }
        // ---- the stream: counted tokens keep their logit for now
#pragma unroll
        for (int k = 0; k < LG_LOADS; k++) {
            const int i = (warp + k * LG_WARPS) * LG_BLOCK;  // the block's place in the chunk
            const int first = token_at(p, t0 + i);
            uint32_t bits = 0;
            if constexpr (VEC) bits = __shfl_sync(0xffffffffu, words, k * 4 + (lane >> 3)) >> (4 * (lane & 7));
            uint32_t c[4] = {};
            if constexpr (COUNT) {
                const int at = t0 - c0 + i;
                if constexpr (!VEC) {
#pragma unroll
                    for (int j = 0; j < 4; j++) c[j] = K::get(counts, at + 32 * j + lane);
                } else if constexpr (SHORT) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(counts + (at + 4 * lane) / 2);
                    c[0] = u.x & 0xFFFFu; c[1] = u.x >> 16; c[2] = u.y & 0xFFFFu; c[3] = u.y >> 16;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4 *>(counts + at + 4 * lane);
                    c[0] = u.x; c[1] = u.y; c[2] = u.z; c[3] = u.w;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int in = VEC ? 4 * lane + j : 32 * j + lane;
                bool allowed;
                if constexpr (VEC) allowed = (bits >> j) & 1u;
                else allowed = (__shfl_sync(0xffffffffu, words, k * 4 + j) >> lane) & 1u;
                if (COUNT && c[j]) {
                    list[atomicAdd(&n_listed[chunk & 1], 1)] = (uint16_t)(i + in);
                } else {
                    if (!allowed) x[k][j] = -INFINITY;
                    if (x[k][j] > best.v && first + in < p.vocab) best = Best{x[k][j], first + in};
                }
            }
            if (!r.dst) continue;
            if constexpr (VEC) {
                const int t = first + 4 * lane;
                if (t + 4 <= p.vocab) {
                    *reinterpret_cast<float4 *>(r.dst + t) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (t + j < p.vocab) r.dst[t + j] = x[k][j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (first + 32 * j + lane < p.vocab) r.dst[first + 32 * j + lane] = x[k][j];
            }
        }
        const bool more = t0 + LG_CHUNK < own;
        if (more) {
            load_chunk<VEC>(p, r.src, t0 + LG_CHUNK, x);
            words = load_words(p, r, t0 + LG_CHUNK);
        }
        // ---- the listed tokens: those without a bias from the list, the others from the bias list
        if constexpr (COUNT) {
            __syncthreads();
            if (tid == 0) n_listed[~chunk & 1] = 0;
            auto settle = [&](int t, uint32_t c, float s) {
                const float v = constrained<SHORT>(p, r, row, t, c, s);
                if (v > best.v || (v == best.v && best.token >= 0 && t < best.token)) best = Best{v, t};
                if (r.dst) r.dst[t] = v;
            };
            const int listed = n_listed[chunk & 1];
            for (int q = tid; q < listed; q += LG_THREADS) {
                const int i = t0 + list[q];
                const uint32_t c = K::get(counts, i - c0);
                if (!(c & K::BIASED)) settle(token_at(p, i), c, 0.0f);
            }
            for (int e = r.b0 + tid; e < r.b1; e += LG_THREADS) {
                const int tok = p.bias_tokens[e], i = place_of(p, tok);
                if (i < t0 || i >= t0 + LG_CHUNK) continue;
                const uint32_t c = K::get(counts, i - c0);
                float s = p.bias_values[e];
                if (c & K::AGAIN) {  // the token's first entry adds up all of them, in order
                    int f = r.b0;
                    while (f < e && p.bias_tokens[f] != tok) f++;
                    if (f < e) continue;
                    for (f = e + 1; f < r.b1; f++)
                        if (p.bias_tokens[f] == tok) s = __fadd_rn(s, p.bias_values[f]);
                }
                settle(tok, c, s);
            }
            if (more) __syncthreads();  // the next stream reuses the list
        }
    }
    return best;
}

// VEC: rows are 16-byte aligned (4 consecutive tokens per load); else one token per load, the warp's consecutive.
// COUNT: the call has histories or biases.
template <bool VEC, bool COUNT>
__global__ void __launch_bounds__(LG_THREADS, 4) logits_kernel(const LogitsParams p) {
    extern __shared__ __align__(16) uint32_t counts[];  // p.count_bytes, then the list
    __shared__ Best warp_best[LG_THREADS / 32];
    __shared__ __align__(8) Best candidate[LG_CLUSTER];  // in the first CTA: every CTA's
    __shared__ __align__(8) uint64_t pushed;
    __shared__ int n_listed[2];
    const int tid = threadIdx.x, C = (int)gridDim.x, rank = (int)blockIdx.x, row = blockIdx.y;
    const bool push = p.choice && C > 1;
    if (COUNT) {
        for (int i = tid; i < p.count_bytes / 16; i += LG_THREADS) reinterpret_cast<uint4 *>(counts)[i] = uint4{0, 0, 0, 0};
        if (tid < 2) n_listed[tid] = 0;
    }
    if (push) {  // the barrier for the candidates, set up before any CTA can arrive on it
        if (rank == 0 && tid == 0) {
            mbar_init(&pushed, (uint32_t)(C - 1));
            fence_barrier_init();
        }
        __syncwarp();
        cluster_arrive();
    }
    grid_dependency_wait();
    grid_dependents_launch();

    // the first logits are under way before anything waits for the lists' offsets
    Row r{};
    r.src = p.logits + (long long)row * p.logits_stride;
    r.dst = p.out ? p.out + (long long)row * p.out_stride : nullptr;
    float x[LG_LOADS][4];
    load_chunk<VEC>(p, r.src, 0, x);
    const bool report = rank == 0 && tid == 0;
    if (p.mask) {
        const int m = p.mask_rows ? p.mask_rows[row] : row;
        r.barred = m < -1 || m >= p.n_mask_rows;
        if (r.barred && report) record_error(p.err, DEVERR_BADLEN);
        if (m >= 0 && !r.barred) r.mask = p.mask + (long long)m * p.mask_stride;
    }
    if (COUNT && p.tokens) {
        const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
        list_range(p.token_offsets, row, p.n_tokens, p.err, report, r.h0, r.h1);
        r.prompt_end = r.h0 + min(max(prompt, 0), r.h1 - r.h0);
    }
    if (COUNT && p.bias_tokens) list_range(p.bias_offsets, row, p.n_bias, p.err, report, r.b0, r.b1);
    uint16_t *list = reinterpret_cast<uint16_t *>(reinterpret_cast<uint8_t *>(counts) + p.count_bytes);
    Best best;
    if (!COUNT || r.h1 - r.h0 <= LG_SHORT)
        best = work_row<VEC, COUNT, true>(p, r, row, p.count_bytes / 2, counts, list, n_listed, x);
    else
        best = work_row<VEC, COUNT, false>(p, r, row, p.count_bytes / 4, counts, list, n_listed, x);

    // ---- the greedy choice
    if (!p.choice) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (push) cluster_wait();  // the first CTA's barrier is set up
    if (tid >= 32) return;
    best = tid < LG_THREADS / 32 ? warp_best[tid] : Best{-INFINITY, -1};
#pragma unroll
    for (int o = LG_THREADS / 64; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    if (C > 1 && rank != 0) {
        if (tid == 0) {
            st_cluster_u32x2(cluster_map(&candidate[rank], 0), __float_as_uint(best.v), (uint32_t)best.token);
            mbar_arrive_remote(cluster_map(&pushed, 0));
        }
        return;
    }
    if (C > 1) {
        // 1 s: the other CTAs of the cluster are resident and only stream their ranges
        const bool ok = mbar_wait_cluster_bounded(&pushed, 0, 1000000000ull, p.err);
        if (!__all_sync(0xffffffffu, ok)) return;
        if (tid > 0) best = tid < C ? candidate[tid] : Best{-INFINITY, -1};
#pragma unroll
        for (int o = LG_CLUSTER / 2; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    }
    if (tid == 0) p.choice[row] = best.token;
}

template <bool VEC, bool COUNT>
int launch_logits(const LogitsParams &p, int cluster, cudaStream_t stream) {
    const size_t smem = COUNT ? p.count_bytes + LG_CHUNK * sizeof(uint16_t) : 0;
    {
        // the shared-memory and cluster-size opt-ins are per-device function attributes
        static std::mutex mu;
        static bool ready[64];
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || dev < 0 || dev >= 64) return fail_cuda(e, "tqk_process_logits: cudaGetDevice");
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(logits_kernel<VEC, COUNT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     LG_COUNT_BYTES_MAX + LG_CHUNK * (int)sizeof(uint16_t));
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(logits_kernel<VEC, COUNT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
    // counts are 29 bits (a token's counter also carries three flags)
    if (a->vocab_size > LG_COUNT_MAX || a->n_tokens > LG_COUNT_MAX)
        return fail(TQK_EUNSUPPORTED, "tqk_process_logits: vocab_size or n_tokens above 2^29 - 1");
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
    // CTAs per row: 8, each with at least 2048 tokens, or 16 while all of them run at once (4 per SM).  128256 tokens
    // with everything on, 16 against 8 CTAs per row: 1 row 9.4 and 14.0 us, 64 rows 39.8 and 30.3 us, 256 rows 168 and 142 us
    const int most = (long long)a->n_rows * LG_CLUSTER <= 4LL * device_info()->sm_count ? LG_CLUSTER : 8;
    while (1 << p.log_c < most && a->vocab_size > 2048 << p.log_c) p.log_c++;
    const int cluster = 1 << p.log_c;
    p.own_blocks = (int)(((int64_t)a->vocab_size + (int64_t)cluster * LG_BLOCK - 1) / ((int64_t)cluster * LG_BLOCK));
    const bool vec = ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 &&
                     (a->n_rows == 1 || ((ls | (p.out ? os : 0)) & 3) == 0);
    const bool count = penal || a->bias_tokens;
    // 16 bits per token of the CTA (a long history's 32 bits take two rounds), whole chunks of 32-bit counters
    const int64_t chunk_bytes = LG_CHUNK * 4, bytes = ((int64_t)p.own_blocks * LG_BLOCK * 2 + chunk_bytes - 1) / chunk_bytes * chunk_bytes;
    p.count_bytes = (int)(bytes < LG_COUNT_BYTES_MAX ? bytes : LG_COUNT_BYTES_MAX);
    cudaStream_t st = (cudaStream_t)stream;
    if (vec) return count ? launch_logits<true, true>(p, cluster, st) : launch_logits<true, false>(p, cluster, st);
    return count ? launch_logits<false, true>(p, cluster, st) : launch_logits<false, false>(p, cluster, st);
}
