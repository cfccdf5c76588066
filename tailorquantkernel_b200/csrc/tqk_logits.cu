// tqk_logits.cu -- constraints on the next token (tqk_process_logits):
// repetition, frequency and presence penalties over each row's history, token
// biases, a grammar's bit mask, and the greedy choice among what is left.
//
// One thread-block cluster per row; blocks of 128 tokens are dealt out to its
// CTAs in turn.  The bulk of a row -- tokens in neither its history nor its bias
// list -- only meets the mask and is streamed through registers: 8 16-byte loads
// in flight per thread, each logit read and written once, which is the kernel's
// floor (8 bytes of DRAM traffic per token).  256 rows of 128256 tokens take 48 us
// with a mask alone (floor 41) and 112 us with histories of 500 to 16000 and biases,
// where issue slots bound it (60% busy).  Around the stream:
//   * while the first logits are on their way, every CTA scans the history and
//     counts its own tokens in shared memory (a counter per token: seen, in the
//     bias list, and the count after the prompt; integer atomics, so their order
//     does not show) and marks them in a bitmap.  Frequent tokens have neighbouring
//     ids in many vocabularies; dealing out small blocks spreads them over the CTAs;
//   * the stream reads the bitmap like a second mask; each warp then lists its
//     marked tokens, fetches their logits again (ahead of the next logits of the
//     stream, or they would queue behind those: 5% of the time with histories) and
//     works the list off with all lanes, so the division and the branches of the
//     penalties cost by the distinct tokens of the history, not by the vocabulary;
//   * each CTA pushes its candidate for the greedy choice to the first CTA's
//     shared memory; a cluster barrier later the first CTA compares them.
#include "tqk_internal.h"
#include "tqk_logits_plan.h"

#include <climits>
#include <mutex>
#include <type_traits>

namespace tqk {
namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_WARPS = LG_THREADS / 32;
constexpr int LG_BLOCK = 128;                            // tokens per block: a warp's 16-byte loads
constexpr int LG_LOADS = 8;                              // blocks per warp and chunk, in registers
constexpr int LG_CHUNK = LG_WARPS * LG_LOADS * LG_BLOCK; // 8192 tokens
constexpr int LG_COUNT_BYTES_MAX = 64 << 10;             // counters per CTA
constexpr int LG_LIST = 256;                             // listed tokens per warp at a time
constexpr int LG_SCAN = 4 * LG_THREADS;                  // history entries staged at a time: a 16-byte copy per thread
constexpr int LG_STAGE = 2 * LG_SCAN;                    // ... and the next ones; later the listed tokens' logits
static_assert(LG_STAGE == LG_WARPS * LG_LIST, "the listed logits take the staging's memory");
// Counters: 16 bits per token (two to a word) for histories with up to LG_SHORT entries behind the prompt, else 32 bits.
// From the top: seen, in the bias list, more than once in the bias list, and the count after the prompt.  The width is
// a value of the row, not of the type: two copies of the row's work in one kernel miss the instruction cache (12% slower
// with short histories).
constexpr int LG_SHORT = (1 << 13) - 1;
constexpr int LG_COUNT_MAX = (1 << 29) - 1;
struct Counters {
    uint32_t *words;
    int half;  // 1: 16 bits, 0: 32 bits
    __device__ __forceinline__ uint32_t seen() const { return half ? 0x8000u : 0x80000000u; }
    __device__ __forceinline__ uint32_t biased() const { return seen() >> 1; }
    __device__ __forceinline__ uint32_t again() const { return seen() >> 2; }
    __device__ __forceinline__ uint32_t count() const { return (seen() >> 2) - 1; }
    // the word of token t, and its counter's place in it
    __device__ __forceinline__ uint32_t *word(int t) const { return words + (t >> half); }
    __device__ __forceinline__ int shift(int t) const { return (t & half) * 16; }
    __device__ __forceinline__ uint32_t get(int t) const { return (*word(t) >> shift(t)) & (seen() * 2 - 1); }
};

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
    int count_bytes;  // counters' shared memory
    int bitmap_bytes; // the bitmap's: whole chunks
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

// 16-byte units of the counters and the bitmap of counted tokens behind them.
__device__ __forceinline__ int zero_units(const LogitsParams &p) { return (p.count_bytes + p.bitmap_bytes) / 16; }

// What all threads of a CTA know of their row.
struct Row {
    const float *src;
    float *dst;
    const uint32_t *mask;  // or nullptr
    bool barred;           // a bad mask row index: nothing is allowed
    int h0, h1, prompt_end, b0, b1;
    Counters counters;
    int span;  // tokens that the counters cover at a time: whole chunks, or all of the CTA's
    float repetition, frequency, presence;
};

// Bit t of the row's mask.
__device__ __forceinline__ bool allowed_token(const Row &r, int t) {
    return !r.barred && (!r.mask || (r.mask[t >> 5] >> (t & 31)) & 1u);
}

// A listed token's final value from its logit v: penalties by its counter c, then its biases' sum s.
__device__ __forceinline__ float constrained(const LogitsParams &p, const Row &r, float v, uint32_t c, float s) {
    const Counters &k = r.counters;
    if (p.repetition && (c & (k.seen() | k.count())))
        v = v > 0.0f ? __fdiv_rn(v, r.repetition) : __fmul_rn(v, r.repetition);
    if (c & k.count()) v = __fsub_rn(__fsub_rn(v, __fmul_rn(r.frequency, __uint2float_rn(c & k.count()))), r.presence);
    return c & k.biased() ? __fadd_rn(v, s) : v;
}

// The CTA's tokens: block b of the row is block b >> log_c of CTA b mod C.  The row's token at place i of them:
__device__ __forceinline__ int token_at(const LogitsParams &p, unsigned i) {
    return (int)((((i / LG_BLOCK) << p.log_c) + blockIdx.x) * LG_BLOCK + i % LG_BLOCK);
}
// ... and the place of token `tok`, or -1 when it is another CTA's or outside the vocabulary.
__device__ __forceinline__ int place_of(const LogitsParams &p, int tok) {
    const unsigned blk = (unsigned)tok / LG_BLOCK;
    const bool own = (blk & ((1u << p.log_c) - 1)) == blockIdx.x && (unsigned)tok < (unsigned)p.vocab;
    return own ? (int)(blk >> p.log_c) * LG_BLOCK + tok % LG_BLOCK : -1;
}

// The logits of the chunk at place t0, 8 blocks per warp.  VEC: tokens 4 lane .. 4 lane + 3 of each block; else tokens
// lane, 32 + lane, 64 + lane, 96 + lane.  Places behind the vocabulary hold 0.
template <bool VEC>
__device__ __forceinline__ void load_chunk(const LogitsParams &p, const float *src, int t0, float (&x)[LG_LOADS][4]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first0 = token_at(p, t0 + warp * LG_BLOCK), step = (LG_WARPS << p.log_c) * LG_BLOCK;
    const float *at = src + first0 + (VEC ? 4 * lane : lane);
#pragma unroll
    for (int k = 0; k < LG_LOADS; k++, at += step) {
        const int left = p.vocab - first0 - k * step;  // tokens from the block's first on
        if (left >= LG_BLOCK) {
            if constexpr (VEC) {
                const float4 f = load_stream(reinterpret_cast<const float4 *>(at));
                x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) x[k][j] = load_stream(at + 32 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int in = VEC ? j : 32 * j;
                x[k][j] = in + (VEC ? 4 * lane : lane) < left ? at[in] : 0.0f;
            }
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
// The bits of this lane's 4 tokens of block k, from words laid out as above.
template <bool VEC>
__device__ __forceinline__ uint32_t lane_bits(uint32_t words, int k) {
    const int lane = threadIdx.x & 31;
    if constexpr (VEC) return (__shfl_sync(0xffffffffu, words, 4 * k + (lane >> 3)) >> (4 * (lane & 7))) & 0xFu;
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) bits |= ((__shfl_sync(0xffffffffu, words, 4 * k + j) >> lane) & 1u) << j;
    return bits;
}

// Adds unit to (ADD) or sets it in a word of shared memory and sets a bit in another, without a branch.
template <bool ADD>
__device__ __forceinline__ void mark_shared(bool go, uint32_t word, uint32_t unit, uint32_t bits, uint32_t bit) {
    if constexpr (ADD)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %0, 0;\n\t@p red.shared.add.u32 [%1], %2;\n\t"
                     "@p red.shared.or.b32 [%3], %4;\n\t}" ::"r"((uint32_t)go), "r"(word), "r"(unit), "r"(bits), "r"(bit)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %0, 0;\n\t@p red.shared.or.b32 [%1], %2;\n\t"
                     "@p red.shared.or.b32 [%3], %4;\n\t}" ::"r"((uint32_t)go), "r"(word), "r"(unit), "r"(bits), "r"(bit)
                     : "memory");
}

// Counts the history's entries among this CTA's tokens [c0, c0 + span) and marks them in the bitmap, once the CTA's
// threads have met (the counters are zero then).  The entries are staged in shared memory, 1024 at a time and the next
// 1024 on their way, so that they take no registers beside the logits.  What bounds this is the instructions issued,
// every CTA of the row looking at every entry (256 rows: 68 M warp instructions, 16 M without histories): each lane
// updates its own entries, one in C active, without a branch.  Collecting the CTA's entries first, to update them with
// all lanes, takes more of them (7% slower).
__device__ __forceinline__ void count_history(const LogitsParams &p, const Row &r, int c0, uint32_t *bitmap, uint32_t *lists) {
    const Counters &k = r.counters;
    const int tid = threadIdx.x;
    const uint32_t staged = smem_u32(lists + 4 * tid);  // this thread's
    // from a 16-byte boundary on; entries before h0 are skipped.  An array that is not 16-byte aligned is copied word by word
    const int wide_end = (reinterpret_cast<uintptr_t>(p.tokens) & 15) == 0 ? min(p.n_tokens - 3, r.h1) : INT_MIN;
    auto fetch = [&](int base, uint32_t to) {
        const int i = base + 4 * tid;
        if (i < wide_end) copy_async_16(to, p.tokens + i);
        else
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < r.h1) copy_async_4(to + 4 * j, p.tokens + i + j);
        copy_async_commit();
    };
    // a token's block is the CTA's when the block's last bits are its rank; the CTA's places below `end` are in the span
    // and in the vocabulary
    const uint32_t rank = blockIdx.x * LG_BLOCK, deal = ((1u << p.log_c) - 1) * LG_BLOCK;
    const int last = (p.vocab - 1) / LG_BLOCK, blocks = (last - (int)blockIdx.x + (1 << p.log_c)) >> p.log_c;
    const bool last_own = ((last * LG_BLOCK) & (int)deal) == (int)rank;
    const int end = min(max(blocks * LG_BLOCK - (last_own ? (last + 1) * LG_BLOCK - p.vocab : 0) - c0, 0), r.span);
    const uint32_t words = smem_u32(k.words), bits = smem_u32(bitmap), seen = k.seen(), to_bytes = 2 - k.half;
    // the entries at base .. base + LG_SCAN - 1 that lie in [from, to), this thread's in v
    auto count = [&](uint4 v, int base, int from, int to, auto made) {
        uint32_t tok[4] = {v.x, v.y, v.z, v.w};
        if (base < from || base + LG_SCAN > to) {
            const int i = base + 4 * tid;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < from || i + j >= to) tok[j] = UINT_MAX;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t t = (((tok[j] >> p.log_c) & ~(LG_BLOCK - 1u)) | (tok[j] & (LG_BLOCK - 1u))) - c0;
            const uint32_t word = words + ((t << to_bytes) & ~3u), unit = (decltype(made)::value ? 1u : seen) << k.shift(t);
            mark_shared<decltype(made)::value>(((tok[j] ^ rank) & deal) == 0 && t < (uint32_t)end, word, unit,
                                               bits + (t >> 5) * 4, __funnelshift_l(0u, 1u, t));
        }
    };
    const int first = r.h0 & ~3;
    fetch(first, staged);
    fetch(first + LG_SCAN, staged + LG_SCAN * 4);
    __syncthreads();
    uint32_t turn = 0;
#pragma unroll 1
    for (int base = first; base < r.h1; base += LG_SCAN, turn ^= LG_SCAN * 4) {
        copy_async_wait<1>();  // each thread reads only what it copied
        const uint4 v = ld_shared_u32x4(staged + turn);
        fetch(base + 2 * LG_SCAN, staged + turn);
        if (base < r.prompt_end) count(v, base, r.h0, r.prompt_end, std::false_type{});
        if (base + LG_SCAN > r.prompt_end && r.prompt_end < r.h1) count(v, base, r.prompt_end, r.h1, std::true_type{});
    }
    copy_async_wait_all();
}

// This CTA's share of a row.  On entry x holds the first chunk, and the counters and their bitmap are zero.
template <bool VEC, bool COUNT>
__device__ __forceinline__ Best work_row(const LogitsParams &p, const Row &r, uint32_t *bitmap, uint32_t *lists,
                                         float (&x)[LG_LOADS][4]) {
    const Counters &counters = r.counters;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int own = p.own_blocks * LG_BLOCK, step = (LG_WARPS << p.log_c) * LG_BLOCK;
    Best top{-INFINITY, -1};   // of the warp's streamed tokens
    Best best{-INFINITY, -1};  // of this thread's listed ones
    // this warp's marked tokens as bits of its words, 32 w + b, and their logits
    uint16_t *list = reinterpret_cast<uint16_t *>(lists + LG_STAGE) + warp * LG_LIST;
    float *list_v = reinterpret_cast<float *>(lists) + warp * LG_LIST;
    uint32_t words = load_words(p, r, 0);
    int c0 = 0;
    auto settle = [&](int t, float v) {
        if (v > best.v || (v == best.v && best.token >= 0 && t < best.token)) best = Best{v, t};
        if (r.dst) r.dst[t] = v;
    };
    // lists marked tokens of the chunk at t0, as many as fit, and takes them out of marks; their logits are on their way
    auto list_marks = [&](uint32_t &marks, int t0) {
        if (!__any_sync(0xffffffffu, marks)) return 0;
        int at = __popc(marks);
        if (__reduce_add_sync(0xffffffffu, at) > LG_LIST) at = min(at, LG_LIST / 32);
        const int n_own = at;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int before = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += before;
        }
        const int n = __shfl_sync(0xffffffffu, at, 31);
        at -= n_own;
        const float *from = r.src + token_at(p, t0 + (warp + (lane >> 2) * LG_WARPS) * LG_BLOCK) + 32 * (lane & 3);
        for (int q = 0; q < n_own; q++, marks &= marks - 1) {
            const int b = __ffs(marks) - 1;
            list[at + q] = (uint16_t)(32 * lane + b);
            copy_async_4(smem_u32(list_v + at + q), from + b);  // in place: still the logit
        }
        return n;
    };
    // the n listed tokens of the chunk at t0, `mask` its mask words; those with a bias are left to the bias list
    auto work_off = [&](int n, uint32_t mask, int t0) {
        copy_async_wait_all();
        __syncwarp();
        for (int q0 = 0; q0 < n; q0 += 32) {
            const unsigned e = q0 + lane < n ? list[q0 + lane] : 0;
            const bool allowed = (__shfl_sync(0xffffffffu, mask, e >> 5) >> (e & 31)) & 1u;
            if (q0 + lane >= n) continue;
            const unsigned i = t0 + (warp + e / LG_BLOCK * LG_WARPS) * LG_BLOCK + e % LG_BLOCK;
            const uint32_t c = counters.get(i - c0);
            if (!(c & counters.biased()))
                settle(token_at(p, i), allowed ? constrained(p, r, list_v[q0 + lane], c, 0.0f) : -INFINITY);
        }
        __syncwarp();
    };
    for (int t0 = 0; t0 < own; t0 += LG_CHUNK) {
        if constexpr (COUNT) {
            if (t0 == 0 || t0 == c0 + r.span) {
                // ---- the counters of the tokens from t0 on
                if (t0 > 0) {
                    __syncthreads();  // the last span's are done with
                    for (int i = tid; i < zero_units(p); i += LG_THREADS)
                        reinterpret_cast<uint4 *>(counters.words)[i] = uint4{0, 0, 0, 0};
                }
                c0 = t0;
                count_history(p, r, c0, bitmap, lists);
                for (int i = r.b0 + tid; i < r.b1; i += LG_THREADS) {
                    const int t = place_of(p, p.bias_tokens[i]) - c0;
                    if ((unsigned)t >= (unsigned)r.span) continue;
                    const uint32_t flag = counters.biased() << counters.shift(t);
                    if (atomicOr(counters.word(t), flag) & flag) atomicOr(counters.word(t), flag >> 1);
                    atomicOr(&bitmap[t >> 5], 1u << (t & 31));
                }
                __syncthreads();
            }
        }
        // ---- the stream: marked tokens keep their logit for now
        uint32_t marks = 0;
        if constexpr (COUNT) marks = bitmap[(t0 - c0 + (warp + (lane >> 2) * LG_WARPS) * LG_BLOCK) / 32 + (lane & 3)];
        const int first0 = token_at(p, t0 + warp * LG_BLOCK);
        float *to = r.dst ? r.dst + first0 + (VEC ? 4 * lane : lane) : nullptr;
#pragma unroll
        for (int k = 0; k < LG_LOADS; k++) {
            const int left = p.vocab - first0 - k * step;  // tokens from the block's first on
            const uint32_t allowed = lane_bits<VEC>(words, k), listed = COUNT ? lane_bits<VEC>(marks, k) : 0u;
            float y[4];  // what is stored
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = ((allowed | listed) >> j) & 1u ? x[k][j] : -INFINITY;
            if (r.dst) {
                float *d = to + k * step;
                if (left >= LG_BLOCK) {
                    if constexpr (VEC) {
                        *reinterpret_cast<float4 *>(d) = make_float4(y[0], y[1], y[2], y[3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) d[32 * j] = y[j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int in = VEC ? j : 32 * j;
                        if (in + (VEC ? 4 * lane : lane) < left) d[in] = y[j];
                    }
                }
            }
            // the warp's best: a block seldom beats all blocks before it, so one vote per block (NaN loses every
            // comparison); when one may, the largest value's first token among those that the stream settles
            if (__any_sync(0xffffffffu, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) > top.v)) {
                float most = -INFINITY;
                unsigned token = UINT_MAX;
#pragma unroll
                for (int j = 3; j >= 0; j--) {
                    const int in = VEC ? 4 * lane + j : 32 * j + lane;
                    if (y[j] >= most && y[j] > top.v && in < left && !((listed >> j) & 1u)) {
                        most = y[j];
                        token = first0 + k * step + in;
                    }
                }
                const int bits = __float_as_int(most + 0.0f);  // -0 as 0
                const int order = token != UINT_MAX ? bits ^ ((bits >> 31) & 0x7FFFFFFF) : INT_MIN;
                const int o = __reduce_max_sync(0xffffffffu, order);
                if (o != INT_MIN) {
                    top.v = __int_as_float(o ^ ((o >> 31) & 0x7FFFFFFF));
                    top.token = (int)__reduce_min_sync(0xffffffffu, order == o ? token : UINT_MAX);
                }
            }
        }
        const uint32_t mask = words;
        int n_listed = 0;
        if constexpr (COUNT) {
            __syncwarp();
            n_listed = list_marks(marks, t0);
        }
        if (t0 + LG_CHUNK < own) {  // the next logits load while the marked tokens are worked off
            load_chunk<VEC>(p, r.src, t0 + LG_CHUNK, x);
            words = load_words(p, r, t0 + LG_CHUNK);
        }
        if constexpr (COUNT) {
            while (n_listed > 0) {  // once, unless there are more than the list holds
                work_off(n_listed, mask, t0);
                n_listed = list_marks(marks, t0);
            }
            // ---- the span's tokens with a bias, once their raw logits are stored
            if (r.b1 > r.b0 && (t0 + LG_CHUNK >= own || t0 + LG_CHUNK == c0 + r.span)) {
                __syncthreads();
                for (int e = r.b0 + tid; e < r.b1; e += LG_THREADS) {
                    const int tok = p.bias_tokens[e], i = place_of(p, tok);
                    if ((unsigned)(i - c0) >= (unsigned)r.span) continue;
                    const uint32_t c = counters.get(i - c0);
                    float s = p.bias_values[e];
                    const float v = r.src[tok];  // in place: still the logit
                    if (c & counters.again()) {  // the token's first entry adds up all of them, in order
                        int f = r.b0;
                        while (f < e && p.bias_tokens[f] != tok) f++;
                        if (f < e) continue;
                        for (f = e + 1; f < r.b1; f++)
                            if (p.bias_tokens[f] == tok) s = __fadd_rn(s, p.bias_values[f]);
                    }
                    settle(tok, allowed_token(r, tok) ? constrained(p, r, v, c, s) : -INFINITY);
                }
            }
        }
    }
    return better(best, top);
}

// VEC: rows are 16-byte aligned (4 consecutive tokens per load); else one token per load, the warp's consecutive.
// COUNT: the call has histories or biases.
template <bool VEC, bool COUNT>
__global__ void __launch_bounds__(LG_THREADS, 4) logits_kernel(const LogitsParams p) {
    extern __shared__ __align__(16) uint32_t counts[];  // p.count_bytes, then the bitmap, then the list
    __shared__ Best warp_best[LG_THREADS / 32];
    __shared__ __align__(8) Best candidate[LG_CLUSTER];  // in the first CTA: every CTA's
    const int tid = threadIdx.x, C = (int)gridDim.x, rank = (int)blockIdx.x, row = blockIdx.y;
    const bool push = p.choice && C > 1;
    if (COUNT) {
        for (int i = tid; i < zero_units(p); i += LG_THREADS) reinterpret_cast<uint4 *>(counts)[i] = uint4{0, 0, 0, 0};
    }
    if (push) cluster_arrive();
    grid_dependency_wait();
    grid_dependents_launch();

    Row r{};
    r.src = p.logits + (long long)row * p.logits_stride;
    r.dst = p.out ? p.out + (long long)row * p.out_stride : nullptr;
    float x[LG_LOADS][4];
    load_chunk<VEC>(p, r.src, 0, x);  // under way before anything waits for the lists' offsets
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
        if (p.repetition) r.repetition = p.repetition[row];
        if (p.frequency) r.frequency = p.frequency[row];
        if (p.presence) r.presence = p.presence[row];
    }
    if (COUNT && p.bias_tokens) list_range(p.bias_offsets, row, p.n_bias, p.err, report, r.b0, r.b1);
    uint32_t *bitmap = counts + p.count_bytes / 4;
    uint32_t *lists = bitmap + p.bitmap_bytes / 4;  // LG_STAGE words, then 16 bits per listed token
    r.counters = Counters{counts, r.h1 - r.prompt_end <= LG_SHORT};
    const int fit = p.count_bytes / (r.counters.half ? 2 : 4);
    r.span = fit >= p.own_blocks * LG_BLOCK ? fit : fit / LG_CHUNK * LG_CHUNK;
    Best best = work_row<VEC, COUNT>(p, r, bitmap, lists, x);

    // ---- the greedy choice
    if (!p.choice) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (push) cluster_wait();  // the first CTA runs, so its shared memory can be written
    if (tid < 32) {
        best = tid < LG_THREADS / 32 ? warp_best[tid] : Best{-INFINITY, -1};
#pragma unroll
        for (int o = LG_THREADS / 64; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
        if (push && rank != 0 && tid == 0)
            st_cluster_u32x2(cluster_map(&candidate[rank], 0), __float_as_uint(best.v), (uint32_t)best.token);
    }
    if (push) {
        // the first CTA must outlast the last push, however long another CTA's share of the lists takes: a barrier of
        // the cluster, not a wait with a time limit
        __syncwarp();
        cluster_sync_all();
    }
    if (rank != 0 || tid >= 32) return;
    if (push) {
        if (tid > 0) best = tid < C ? candidate[tid] : Best{-INFINITY, -1};
#pragma unroll
        for (int o = LG_CLUSTER / 2; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.token, o)});
    }
    if (tid == 0) p.choice[row] = best.token;
}

// What shared memory takes is lost for loads in flight, in steps: 4 CTAs of 47 KB (32 KB of counters) leave 60 KB of L1,
// 4 CTAs of 51 KB only 28 KB (256 rows of 128256 tokens: 111 and 121 us).
size_t logits_smem(int count_bytes, int bitmap_bytes) { return count_bytes + bitmap_bytes + LG_STAGE * 4 + LG_WARPS * LG_LIST * 2; }

// Sets up the kernel on the current device, once: the shared-memory and cluster-size opt-ins are per-device function
// attributes.  *most: CTAs per row, 16 where the device holds such a cluster (a part of a device may not), else 8.
template <bool VEC, bool COUNT>
int prepare_logits(int *most) {
    constexpr auto kernel = logits_kernel<VEC, COUNT>;
    static std::mutex mu;
    static int most_by[64];  // 0 = not set up
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return fail_cuda(e, "tqk_process_logits: cudaGetDevice");
    std::lock_guard<std::mutex> lock(mu);
    if (!most_by[dev]) {
        const int smem = (int)logits_smem(LG_COUNT_BYTES_MAX, LG_COUNT_BYTES_MAX / 16);
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return fail_cuda(e, "tqk_process_logits: kernel attributes");
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        int n = 0;
        if (e == cudaSuccess) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(LG_CLUSTER, 1, 1);
            cfg.blockDim = dim3(LG_THREADS);
            cfg.dynamicSmemBytes = COUNT ? smem : 0;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = LG_CLUSTER;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        }
        if (e != cudaSuccess) (void)cudaGetLastError();  // not an error of the call: smaller clusters
        most_by[dev] = e == cudaSuccess && n > 0 ? LG_CLUSTER : LG_CLUSTER_PORTABLE;
    }
    *most = most_by[dev];
    return TQK_OK;
}

template <bool VEC, bool COUNT>
int launch_logits(const LogitsParams &p, int cluster, cudaStream_t stream) {
    const size_t smem = COUNT ? logits_smem(p.count_bytes, p.bitmap_bytes) : 0;
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
    const bool vec = ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 &&
                     (a->n_rows == 1 || ((ls | (p.out ? os : 0)) & 3) == 0);
    const bool count = penal || a->bias_tokens;
    int most = 0;
    rc = vec ? count ? prepare_logits<true, true>(&most) : prepare_logits<true, false>(&most)
             : count ? prepare_logits<false, true>(&most) : prepare_logits<false, false>(&most);
    if (rc) return rc;
    p.log_c = logits_cluster_log(a->n_rows, a->vocab_size, device_info()->sm_count, most);
    const int cluster = 1 << p.log_c;
    p.own_blocks = (int)(((int64_t)a->vocab_size + (int64_t)cluster * LG_BLOCK - 1) / ((int64_t)cluster * LG_BLOCK));
    // 32 bits per token of the CTA where one chunk holds them all, else 16 and at least a chunk of 32 (a long history's
    // counters take more rounds)
    const int64_t own = (int64_t)p.own_blocks * LG_BLOCK, bytes = own <= LG_CHUNK ? own * 4 : own * 2;
    p.count_bytes = (int)(bytes < LG_COUNT_BYTES_MAX ? bytes : LG_COUNT_BYTES_MAX);
    if (own > LG_CHUNK && p.count_bytes < LG_CHUNK * 4) p.count_bytes = LG_CHUNK * 4;
    const int64_t covered = own < LG_COUNT_BYTES_MAX / 2 ? own : LG_COUNT_BYTES_MAX / 2;
    p.bitmap_bytes = (int)((covered + LG_CHUNK - 1) / LG_CHUNK * (LG_CHUNK / 8));
    cudaStream_t st = (cudaStream_t)stream;
    if (vec) return count ? launch_logits<true, true>(p, cluster, st) : launch_logits<true, false>(p, cluster, st);
    return count ? launch_logits<false, true>(p, cluster, st) : launch_logits<false, false>(p, cluster, st);
}
