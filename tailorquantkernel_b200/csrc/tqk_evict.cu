// tqk_evict.cu -- eviction from Q8 caches by accumulated attention weight
// (tqk_evict_q8).
//
// Each (item, kv head) keeps the `budget` best of its n rows; the j-th kept row
// from slot `budget` on moves into the j-th evicted slot below it.  Every row
// that moves is read at or above slot `budget` and written below it, so moves
// never touch each other's rows and need no order, and no row moves that does
// not have to: about budget * (n - budget) / n rows of a cache cut to `budget`,
// one row of a cache that is one row over.
//
// One thread-block cluster per (item, kv head), a contiguous part of the slots
// per CTA:
//   1. keys: the rank of a row as 32 bits that compare unsigned (protected rows
//      above every weight), into shared memory;
//   2. the budget-th largest key by radix select, 11 + 11 + 10 bits: a histogram
//      per CTA in shared memory, summed over the cluster through distributed
//      shared memory, searched by every CTA alike;
//   3. each thread marks the holes (evicted, below `budget`) and movers (kept,
//      from `budget` on) of its own run of consecutive slots; block and cluster
//      prefix sums of their counts give every one its rank, and their slots go
//      into a list that overwrites the keys;
//   4. the moves are dealt out evenly over the cluster's CTAs, which look up the
//      j-th hole and the j-th mover in the CTAs' lists and copy the rows.
// Only integer counts are summed, so results do not depend on timing.
#include "tqk_internal.h"

#include <climits>
#include <mutex>
#include <type_traits>

namespace tqk {
namespace {

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;                   // histogram bins: digits of 11, 11 and 10 bits
constexpr int EV_BPT = EV_BINS / EV_THREADS;    // bins per thread
constexpr int EV_RUN_MAX = 63;                  // slots per thread: a bit each of a 64-bit mask, an odd number
constexpr int EV_CLUSTER_MAX = 16;
constexpr int EV_BATCH = 128;                   // moves looked up at a time
static_assert(EV_CLUSTER_MAX * EV_THREADS * EV_RUN_MAX == TQK_EVICT_MAX_LEN, "documented limit");

struct EvictParams {
    uint8_t *k, *v;
    long long item_stride;  // bytes
    int n_kv, max_tokens;
    const int *lens;
    int len0, len_step, len_cap;
    int budget, n_first, n_recent;
    const float *weight;
    float *weight_out;
    const int *position;
    int *position_out;
    long long stat_stride;
    int run;  // slots per thread at the longest length
    int *err;
};

struct EvictShared {
    unsigned hist[3][EV_BINS];
    int warp_tot[EV_WARPS];
    int max_pos;             // this CTA's largest position
    int counts[2];           // this CTA's holes and movers
    int ties;                // this CTA's keys equal to the threshold
    unsigned found_bin;
    int found_above;
    int found_count;
    int pre_h[EV_CLUSTER_MAX + 1], pre_m[EV_CLUSTER_MAX + 1];
    int src[EV_BATCH], dst[EV_BATCH];
};

// A float's bits reordered so that unsigned comparison orders them: negative numbers below positive ones,
// -0 as +0, every NaN 0 (below -inf, which becomes 0x007FFFFF).
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (isnan(w)) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t KEY_PROTECTED = 0xFFFFFFFFu;  // above +inf's 0xFF800000

// Exclusive prefix sum of v over the CTA's threads; *total receives the sum.  Ends with a barrier.
__device__ __forceinline__ int block_prefix(int v, int *warp_tot, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < EV_WARPS; w++) {
        const int x = warp_tot[w];
        if (w < warp) before += x;
        all += x;
    }
    __syncthreads();
    *total = all;
    return before + incl - v;
}

// Copies moves [0, n) of sh.src / sh.dst: whole rows of both planes.
template <int NB>
__device__ __forceinline__ void copy_rows(uint8_t *kh, uint8_t *vh, const EvictShared &sh, int n) {
    constexpr int ROW = NB * BLOCK_BYTES;
    using Unit = typename std::conditional<NB % 4 == 0, uint4, uint32_t>::type;  // rows of 4 blocks are 16-byte aligned
    constexpr int UNITS = ROW / (int)sizeof(Unit);
    constexpr int IN_FLIGHT = 4;
    const int total = n * 2 * UNITS;
    for (int i0 = threadIdx.x; i0 < total; i0 += IN_FLIGHT * EV_THREADS) {
        Unit x[IN_FLIGHT];
        Unit *to[IN_FLIGHT];
#pragma unroll
        for (int q = 0; q < IN_FLIGHT; q++) {
            const int i = i0 + q * EV_THREADS;
            if (i >= total) break;
            const int row = i / UNITS, u = i - row * UNITS, m = row >> 1;
            uint8_t *plane = row & 1 ? vh : kh;
            x[q] = reinterpret_cast<const Unit *>(plane + (long long)sh.src[m] * ROW)[u];
            to[q] = reinterpret_cast<Unit *>(plane + (long long)sh.dst[m] * ROW) + u;
        }
#pragma unroll
        for (int q = 0; q < IN_FLIGHT; q++)
            if (i0 + q * EV_THREADS < total) *to[q] = x[q];
    }
}

template <int NB>
__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t keys[];  // [EV_THREADS * run], then the slots of holes and movers
    __shared__ EvictShared sh;
    grid_dependency_wait();
    grid_dependents_launch();
    const int tid = threadIdx.x, C = (int)gridDim.x, rank = (int)blockIdx.x;
    const int kvh = blockIdx.y, item = blockIdx.z;
    int len = p.lens ? p.lens[item] : p.len0 + item * p.len_step;
    if (len < 0 || len > p.len_cap) {
        if (tid == 0) record_error(p.err, DEVERR_BADLEN);
        len = len < 0 ? 0 : p.len_cap;
    }
    const long long at = (long long)item * p.stat_stride + (long long)kvh * p.max_tokens;
    const float *w_in = p.weight + at;
    float *w_out = p.weight_out + at;
    const int *pos_in = p.position ? p.position + at : nullptr;
    int *pos_out = p.position ? p.position_out + at : nullptr;
    const bool copy_w = w_out != w_in, copy_pos = pos_out != pos_in;
    const int budget = p.budget;
    // this CTA's slots [s0, s1), `run` consecutive ones per thread; an odd run keeps the threads' shared-memory
    // words in different banks
    const int per = (len + C * EV_THREADS - 1) / (C * EV_THREADS);
    const int run = per | 1;
    const int s0 = min(len, rank * run * EV_THREADS), s1 = min(len, s0 + run * EV_THREADS), n_own = s1 - s0;
    auto cluster_barrier = [&]() {
        if (C > 1) cluster_sync_all();
        else __syncthreads();
    };

    if (len <= budget) {  // nothing to evict (the same for every CTA of the cluster)
        for (int i = s0 + tid; i < s1; i += EV_THREADS) {
            if (copy_w) w_out[i] = w_in[i];
            if (copy_pos) pos_out[i] = pos_in[i];
        }
        return;
    }

    // ---- 1. keys
    for (int i = tid; i < 3 * EV_BINS; i += EV_THREADS) (&sh.hist[0][0])[i] = 0;
    int newest = 0;
    if (p.n_recent > 0) {
        int m = INT_MIN;
        for (int i = s0 + tid; i < s1; i += EV_THREADS) m = max(m, pos_in[i]);
        m = __reduce_max_sync(0xffffffffu, m);
        if ((tid & 31) == 0) sh.warp_tot[tid >> 5] = m;
        __syncthreads();
        if (tid < 32) {
            m = __reduce_max_sync(0xffffffffu, tid < EV_WARPS ? sh.warp_tot[tid] : INT_MIN);
            if (tid == 0) sh.max_pos = m;
        }
        cluster_barrier();
        newest = INT_MIN;
        for (int r = 0; r < C; r++)
            newest = max(newest, C > 1 ? (int)ld_cluster_u32(cluster_map(&sh.max_pos, r)) : sh.max_pos);
    }
    const long long recent_from = (long long)newest - p.n_recent;  // positions above are protected
    for (int i = tid; i < n_own; i += EV_THREADS) {
        const int s = s0 + i;
        const float w = w_in[s];
        uint32_t key = weight_key(w);
        if (pos_in) {
            const int pos = pos_in[s];
            if (pos < p.n_first || (p.n_recent > 0 && pos > recent_from)) key = KEY_PROTECTED;
            if (copy_pos && s < budget) pos_out[s] = pos;
        }
        if (copy_w && s < budget) w_out[s] = w;
        keys[i] = key;
    }
    __syncthreads();

    // ---- 2. the budget-th largest key: `prefix` holds its digits found so far, `need` of the keys that share
    //         them are kept
    uint32_t prefix = 0;
    int need = budget, equal = 0;
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const int bins = 1 << bits;
        unsigned *hist = sh.hist[pass];
        for (int i = tid; i < n_own; i += EV_THREADS) {
            const uint32_t key = keys[i];
            if (pass == 0 || (key >> (shift + bits)) == (prefix >> (shift + bits)))
                atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        cluster_barrier();
        // thread `tid` counts the bins from the top: descending order, EV_BPT (half as many in the last pass) each
        const int bpt = bins / EV_THREADS;
        int cnt[EV_BPT], sum = 0;
#pragma unroll
        for (int q = 0; q < EV_BPT; q++) {
            cnt[q] = 0;
            if (q < bpt) {
                const int bin = bins - 1 - (tid * bpt + q);
                if (C == 1) cnt[q] = (int)hist[bin];
                else
                    for (int r = 0; r < C; r++) cnt[q] += (int)ld_cluster_u32(cluster_map(&hist[bin], r));
            }
            sum += cnt[q];
        }
        int all, above = block_prefix(sum, sh.warp_tot, &all);
#pragma unroll
        for (int q = 0; q < EV_BPT; q++) {
            if (q < bpt && above < need && need <= above + cnt[q]) {
                sh.found_bin = (unsigned)(bins - 1 - (tid * bpt + q));
                sh.found_above = above;
                sh.found_count = cnt[q];
            }
            above += cnt[q];
        }
        __syncthreads();
        prefix |= sh.found_bin << shift;
        need -= sh.found_above;
        equal = sh.found_count;
        __syncthreads();
    }

    // ---- 3. holes and movers of this thread's run
    const int r0 = tid * run, r1 = min(n_own, r0 + run);
    int tie_rank = 0;  // of this thread's first key equal to the threshold, over the cluster
    if (equal > need) {
        int ties = 0, all;
        for (int i = r0; i < r1; i++) ties += keys[i] == prefix;
        tie_rank = block_prefix(ties, sh.warp_tot, &all);
        if (tid == 0) sh.ties = all;
        cluster_barrier();
        for (int r = 0; r < rank; r++) tie_rank += (int)ld_cluster_u32(cluster_map(&sh.ties, r));
    }
    unsigned long long holes = 0, movers = 0;
    for (int i = r0; i < r1; i++) {
        const uint32_t key = keys[i];
        bool keep = key > prefix;
        if (key == prefix) keep = equal <= need || tie_rank++ < need;
        const unsigned long long bit = 1ull << (i - r0);
        if (s0 + i < budget) holes |= keep ? 0ull : bit;
        else movers |= keep ? bit : 0ull;
    }
    // at most 16 * 63 slots per warp and 32256 per CTA: both counts fit in half a word
    int all;
    const int at2 = block_prefix((__popcll(holes) << 16) | __popcll(movers), sh.warp_tot, &all);
    int *list = reinterpret_cast<int *>(keys);  // every key is read: holes from the front, movers from the back
    const int last = EV_THREADS * run - 1;
    for (int j = at2 >> 16; holes; holes &= holes - 1) list[j++] = s0 + r0 + __ffsll(holes) - 1;
    for (int j = at2 & 0xFFFF; movers; movers &= movers - 1) list[last - j++] = s0 + r0 + __ffsll(movers) - 1;
    if (tid == 0) {
        sh.counts[0] = all >> 16;
        sh.counts[1] = all & 0xFFFF;
    }
    cluster_barrier();
    if (tid == 0) {
        int h = 0, m = 0;
        for (int r = 0; r < C; r++) {
            sh.pre_h[r] = h;
            sh.pre_m[r] = m;
            h += C > 1 ? (int)ld_cluster_u32(cluster_map(&sh.counts[0], r)) : sh.counts[0];
            m += C > 1 ? (int)ld_cluster_u32(cluster_map(&sh.counts[1], r)) : sh.counts[1];
        }
        sh.pre_h[C] = h;
        sh.pre_m[C] = m;
    }
    __syncthreads();

    // ---- 4. this CTA's share of the moves (holes and movers are equally many)
    const long long n_moves = sh.pre_m[C];
    const int m0 = (int)(n_moves * rank / C), m1 = (int)(n_moves * (rank + 1) / C);
    const long long head_off = (long long)item * p.item_stride + (long long)kvh * p.max_tokens * (NB * BLOCK_BYTES);
    for (int b = m0; b < m1; b += EV_BATCH) {
        const int n = min(EV_BATCH, m1 - b);
        if (tid < 2 * n) {
            // the first n threads look up the holes, the next n the movers
            const bool mover = tid >= n;
            const int j = b + (mover ? tid - n : tid);
            const int *pre = mover ? sh.pre_m : sh.pre_h;
            int r = 0;
            while (r + 1 < C && pre[r + 1] <= j) r++;
            const int *slot = mover ? &list[last - (j - pre[r])] : &list[j - pre[r]];
            const int v = C > 1 ? (int)ld_cluster_u32(cluster_map(slot, r)) : *slot;
            (mover ? sh.src : sh.dst)[j - b] = v;
        }
        __syncthreads();
        if (tid < n) {
            w_out[sh.dst[tid]] = w_in[sh.src[tid]];
            if (pos_in) pos_out[sh.dst[tid]] = pos_in[sh.src[tid]];
        }
        copy_rows<NB>(p.k + head_off, p.v + head_off, sh, n);
        __syncthreads();
    }
    if (C > 1) cluster_sync_all();  // no CTA leaves while another reads its list
}

// lens_out[i] = min(len_i, budget), after the eviction has read every length.
__global__ void evict_lens_kernel(const int *lens, int len0, int len_step, int len_cap, int budget, int n, int *out) {
    grid_dependency_wait();
    grid_dependents_launch();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) out[i] = min(min(max(lens ? lens[i] : len0 + i * len_step, 0), len_cap), budget);
}

template <int NB>
int launch_evict(const EvictParams &p, int cluster, dim3 grid, cudaStream_t stream) {
    const size_t smem = (size_t)EV_THREADS * p.run * sizeof(uint32_t);
    // the shared-memory and cluster-size opt-ins are per-device function attributes
    static std::mutex mu;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return fail_cuda(e, "tqk_evict_q8: cudaGetDevice");
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(evict_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     EV_THREADS * EV_RUN_MAX * (int)sizeof(uint32_t));
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(evict_kernel<NB>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return fail_cuda(e, "tqk_evict_q8: kernel attributes");
            ready[dev] = true;
        }
    }
    if (cluster == 1) return launch_pdl(evict_kernel<NB>, grid, dim3(EV_THREADS), smem, stream, p);
    return launch_pdl_cluster(evict_kernel<NB>, grid, dim3(EV_THREADS), smem, stream, (unsigned)cluster, p);
}

}  // namespace
}  // namespace tqk

using namespace tqk;

extern "C" int tqk_evict_q8(const tqk_evict_args *a, tqk_stream_t stream) {
    if (!a) return fail(TQK_EINVAL, "tqk_evict_q8: NULL args");
    if (a->n_items <= 0 || a->n_kv_heads <= 0 || a->head_dim <= 0 || a->max_tokens <= 0)
        return fail(TQK_EINVAL, "tqk_evict_q8: non-positive shape");
    if (a->head_dim % QK) return fail(TQK_EINVAL, "tqk_evict_q8: head_dim % 32 != 0");
    const int nb = a->head_dim / QK;
    if (nb != 1 && nb != 2 && nb != 4 && nb != 8)
        return fail(TQK_EUNSUPPORTED, "tqk_evict_q8: head_dim must be 32, 64, 128 or 256");
    if (a->n_items > 65535 || a->n_kv_heads > 65535) return fail(TQK_EINVAL, "tqk_evict_q8: n_items or n_kv_heads > 65535");
    if (!a->k || !a->v || !a->weight || !a->weight_out) return fail(TQK_EINVAL, "tqk_evict_q8: NULL pointer");
    if (a->budget < 1 || a->budget > a->max_tokens) return fail(TQK_EINVAL, "tqk_evict_q8: budget outside [1, max_tokens]");
    if (a->n_first < 0 || a->n_recent < 0 || (long long)a->n_first + a->n_recent > a->budget)
        return fail(TQK_EINVAL, "tqk_evict_q8: n_first and n_recent must fit in the budget");
    if ((a->position == nullptr) != (a->position_out == nullptr))
        return fail(TQK_EINVAL, "tqk_evict_q8: position and position_out go together");
    if (!a->position && (a->n_first || a->n_recent))
        return fail(TQK_EINVAL, "tqk_evict_q8: n_first and n_recent need positions");
    const long long rows = (long long)a->n_kv_heads * a->max_tokens;
    if (a->n_items > 1 && (a->item_stride < rows * nb || a->stat_item_stride < rows))
        return fail(TQK_EINVAL, "tqk_evict_q8: item_stride or stat_item_stride below one item's rows");
    int max_len;
    if (a->lens) {
        max_len = a->max_len;
        if (max_len < 0 || max_len > a->max_tokens) return fail(TQK_EINVAL, "tqk_evict_q8: max_len outside [0, max_tokens]");
    } else {
        const long long first = a->len0, last = a->len0 + (long long)(a->n_items - 1) * a->len_step;
        const long long lo = first < last ? first : last, hi = first < last ? last : first;
        if (lo < 0 || hi > a->max_tokens) return fail(TQK_EPOS, "tqk_evict_q8: length outside [0, max_tokens]");
        max_len = (int)hi;
    }
    if (max_len > TQK_EVICT_MAX_LEN) return fail(TQK_EUNSUPPORTED, "tqk_evict_q8: lengths above TQK_EVICT_MAX_LEN");
    const uintptr_t planes = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                             (a->n_items > 1 ? (uintptr_t)(a->item_stride * BLOCK_BYTES) : 0);
    if (planes & (nb % 4 == 0 ? 15 : 3))
        return fail(TQK_EALIGN, "tqk_evict_q8: planes and item stride must be 16-byte aligned (4-byte for head_dim 32, 64)");
    if ((reinterpret_cast<uintptr_t>(a->weight) | reinterpret_cast<uintptr_t>(a->weight_out) |
         reinterpret_cast<uintptr_t>(a->position) | reinterpret_cast<uintptr_t>(a->position_out) |
         reinterpret_cast<uintptr_t>(a->lens) | reinterpret_cast<uintptr_t>(a->lens_out)) & 3)
        return fail(TQK_EALIGN, "tqk_evict_q8: sums, positions and lengths must be 4-byte aligned");
    int rc = ensure_device();
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (max_len > 0) {
        EvictParams p{};
        p.k = reinterpret_cast<uint8_t *>(a->k);
        p.v = reinterpret_cast<uint8_t *>(a->v);
        p.item_stride = a->item_stride * BLOCK_BYTES;
        p.n_kv = a->n_kv_heads;
        p.max_tokens = a->max_tokens;
        p.lens = a->lens;
        p.len0 = a->len0;
        p.len_step = a->len_step;
        p.len_cap = max_len;
        p.budget = a->budget;
        p.n_first = a->n_first;
        p.n_recent = a->n_recent;
        p.weight = a->weight;
        p.weight_out = a->weight_out;
        p.position = a->position;
        p.position_out = a->position_out;
        p.stat_stride = a->stat_item_stride;
        p.err = device_info()->err_word;
        // CTAs per (item, head): a portable cluster of 8 for lengths that need more than one CTA's 8192 slots,
        // 16 where 8 do not hold the keys
        int cluster = (max_len + 8191) / 8192;
        if (cluster > 8) cluster = max_len > 8 * EV_THREADS * EV_RUN_MAX ? EV_CLUSTER_MAX : 8;
        p.run = ((max_len + cluster * EV_THREADS - 1) / (cluster * EV_THREADS)) | 1;
        const dim3 grid((unsigned)cluster, (unsigned)a->n_kv_heads, (unsigned)a->n_items);
        switch (nb) {
            case 1: rc = launch_evict<1>(p, cluster, grid, st); break;
            case 2: rc = launch_evict<2>(p, cluster, grid, st); break;
            case 4: rc = launch_evict<4>(p, cluster, grid, st); break;
            default: rc = launch_evict<8>(p, cluster, grid, st); break;
        }
        if (rc) return rc;
    }
    if (!a->lens_out) return TQK_OK;
    return launch_pdl(evict_lens_kernel, dim3((unsigned)((a->n_items + 255) / 256)), dim3(256), 0, st, a->lens, a->len0,
                      a->len_step, max_len, a->budget, a->n_items, a->lens_out);
}
