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
// One thread-block cluster per (item, kv head) -- several where SMs are left
// over, which share step 4 -- a contiguous part of the slots per CTA:
//   1. keys: the rank of a row as 32 bits that compare unsigned (protected rows
//      above every weight), into shared memory;
//   2. the budget-th largest key by radix select, 11 + 11 + 10 bits: a histogram
//      per CTA in shared memory, summed over the cluster through distributed
//      shared memory, searched by every CTA alike.  The second pass lists the keys
//      that share the first digit, and the third only looks at those;
//   3. each thread marks the holes (evicted, below `budget`) and movers (kept,
//      from `budget` on) of its own run of consecutive slots; block and cluster
//      prefix sums of their counts give every one its rank, and their slots go
//      into a list that overwrites the keys;
//   4. the moves are dealt out evenly over the cluster's CTAs, which look up the
//      j-th hole and the j-th mover in the CTAs' lists and copy the rows; every warp
//      works on moves of its own, 4 of them in flight.
// Only integer counts are summed, so results do not depend on timing.
#include "tqk_internal.h"

#include <climits>
#include <mutex>
#include <type_traits>

namespace tqk {
namespace {

constexpr int EV_THREADS = 512;                 // per CTA; EV_WIDE where a long length has an SM for every CTA
constexpr int EV_WIDE = 1024;
constexpr int EV_BINS = 2048;                   // histogram bins: digits of 11, 11 and 10 bits
constexpr int EV_RUN_MAX = 63;                  // slots per thread: a bit each of a 64-bit mask, an odd number
constexpr int EV_CLUSTER_MAX = 8;               // the portable cluster size
constexpr int EV_UNITS = 4;                     // units in flight per thread; a ragged batch, 2, 4, 8: 127, 105, 118 us
constexpr int EV_LOADS = 8;                     // sums and positions in flight per thread
constexpr int EV_ALONE = 100 << 10;             // dynamic shared memory that leaves no room for a second CTA
constexpr int EV_KEY_BYTES_MAX = 140 << 10;     // dynamic shared memory at the longest length
constexpr int EV_NARROW = 1024;                 // slots per CTA where every CTA has an SM
constexpr int EV_PARTS_MAX = 8;                 // clusters per (item, kv head)
constexpr int EV_PARTS_MOVES = 4096;            // from so many moves on
constexpr int EV_STAGE = 8192;                  // slots per CTA whose positions are staged in shared memory
static_assert(EV_CLUSTER_MAX * EV_THREADS * EV_RUN_MAX == TQK_EVICT_MAX_LEN, "documented limit");

struct EvictParams {
    uint8_t *k, *v;
    long long item_stride;  // bytes
    int max_tokens;
    const int *lens;
    int len0, len_step, len_cap;
    int budget, n_first, n_recent;
    const float *weight;
    float *weight_out;
    const int *position;
    int *position_out;
    long long stat_stride;
    int run;        // slots per thread at the longest length
    int staged;     // whether positions are staged: the keys take at most EV_STAGE slots per CTA
    int *lens_out;  // written here unless it aliases lens, else nullptr
    int *err;
};

template <int T>
struct EvictShared {
    __align__(16) unsigned hist[3][EV_BINS];
    int warp_tot[5][T / 32];   // of each block_prefix: a buffer of its own saves a barrier
    int max_pos;                 // this CTA's largest position
    int counts[2];               // this CTA's holes and movers
    int ties;                    // this CTA's keys equal to the threshold
    int n_close;                 // keys that share the first digit
    int found[3][3];             // per digit: the bin of the budget-th key, how many keys lie above it, its own
    int pre_h[EV_CLUSTER_MAX + 1], pre_m[EV_CLUSTER_MAX + 1];
};

// A float's bits reordered so that unsigned comparison orders them: negative numbers below positive ones,
// -0 as +0, every NaN 0 (below -inf, which becomes 0x007FFFFF).
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (isnan(w)) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t KEY_PROTECTED = 0xFFFFFFFFu;  // above +inf's 0xFF800000

// Exclusive prefix sum of v over the CTA's threads; *total receives the sum.  warp_tot: a buffer that no other call uses.
template <int T>
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
    // the warps' totals, one per lane
    int before = lane < T / 32 ? warp_tot[lane] : 0, all = before;
    if (lane >= warp) before = 0;
    before = __reduce_add_sync(0xffffffffu, before);
    *total = __reduce_add_sync(0xffffffffu, all);
    return before + incl - v;
}

// One warp moves rows of both planes from slots src to slots dst, lane l's move in its src and dst, the first n lanes'.
// A row is 9 16-byte units (9 words for head_dim 32), or twice as many; K's and V's units lie next to each other in the
// lanes where both fit, so a lane's place in the row never changes and a move costs one load and one store.  Denser
// layouts (every lane at work, twice the bytes in flight) were slower by 8% for a ragged batch.
template <int NB>
__device__ __forceinline__ void move_rows(uint8_t *kh, uint8_t *vh, int src, int dst, int n) {
    constexpr int ROW = NB * BLOCK_BYTES;
    using Unit = typename std::conditional<NB % 4 == 0, uint4, uint32_t>::type;  // rows of 4 blocks are 16-byte aligned
    constexpr int UNITS = ROW / (int)sizeof(Unit);   // 9 or 18
    constexpr int LOADS = UNITS == 9 ? 1 : 2;        // per move
    constexpr int MOVES = EV_UNITS / LOADS;          // in flight
    const int lane = threadIdx.x & 31;
    const bool active = lane < 18;
    uint8_t *base[LOADS];
#pragma unroll
    for (int l = 0; l < LOADS; l++)
        base[l] = LOADS == 2 ? (l ? vh : kh) + lane * sizeof(Unit)
                             : lane < 9 ? kh + lane * sizeof(Unit) : vh + (lane - 9) * sizeof(Unit);
    for (int m0 = 0; m0 < n; m0 += MOVES) {
        Unit x[MOVES][LOADS];
#pragma unroll
        for (int q = 0; q < MOVES; q++) {
            const long long from = (long long)__shfl_sync(0xffffffffu, src, m0 + q) * ROW;
#pragma unroll
            for (int l = 0; l < LOADS; l++)
                if (active && m0 + q < n) x[q][l] = *reinterpret_cast<const Unit *>(base[l] + from);
        }
#pragma unroll
        for (int q = 0; q < MOVES; q++) {
            const long long to = (long long)__shfl_sync(0xffffffffu, dst, m0 + q) * ROW;
#pragma unroll
            for (int l = 0; l < LOADS; l++)
                if (active && m0 + q < n) *reinterpret_cast<Unit *>(base[l] + to) = x[q][l];
        }
    }
}

// PARTS: several clusters share an (item, kv head)'s moves.
template <int NB, int T, bool PARTS>
__global__ void __launch_bounds__(T, 1024 / T) evict_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t keys[];  // [T * run], then the slots of holes and movers
    __shared__ EvictShared<T> sh;
    const int tid = threadIdx.x, C = PARTS ? EV_CLUSTER_MAX : (int)gridDim.x;
    const int rank = PARTS ? (int)blockIdx.x % EV_CLUSTER_MAX : (int)blockIdx.x;
    const int part = PARTS ? (int)blockIdx.x / EV_CLUSTER_MAX : 0, parts = PARTS ? (int)gridDim.x / EV_CLUSTER_MAX : 1;
    for (int i = tid; i < 3 * EV_BINS / 4; i += T) reinterpret_cast<uint4 *>(sh.hist)[i] = uint4{0, 0, 0, 0};
    if (tid == 0) {
        sh.max_pos = INT_MIN;
        sh.n_close = 0;
    }
    __syncthreads();
    grid_dependency_wait();
    grid_dependents_launch();
    const int kvh = blockIdx.y, item = blockIdx.z;
    int len = p.lens ? p.lens[item] : p.len0 + item * p.len_step;
    if (len < 0 || len > p.len_cap) {
        if (tid == 0) record_error(p.err, DEVERR_BADLEN);
        len = len < 0 ? 0 : p.len_cap;
    }
    const int budget = p.budget;
    if (p.lens_out && blockIdx.x == 0 && kvh == 0 && tid == 0) p.lens_out[item] = min(len, budget);
    const long long at = (long long)item * p.stat_stride + (long long)kvh * p.max_tokens;
    const float *w_in = p.weight + at;
    float *w_out = p.weight_out + at;
    const int *pos_in = p.position ? p.position + at : nullptr;
    int *pos_out = p.position ? p.position_out + at : nullptr;
    const bool copy_w = part == 0 && w_out != w_in, copy_pos = part == 0 && pos_out != pos_in;
    // this CTA's slots [s0, s1), `run` consecutive ones per thread; an odd run keeps the threads' shared-memory
    // words in different banks
    const int run = ((len + C * T - 1) / (C * T)) | 1;
    const int s0 = min(len, rank * run * T), s1 = min(len, s0 + run * T), n_own = s1 - s0;
    auto cluster_barrier = [&]() {
        __syncthreads();  // the cluster barrier's instructions meet converged warps
        if (C > 1) cluster_sync_all();
    };

    if (len <= budget) {  // nothing to evict (the same for every CTA of the cluster)
        for (int i = s0 + tid; i < s1; i += T) {
            if (copy_w) w_out[i] = w_in[i];
            if (copy_pos) pos_out[i] = pos_in[i];
        }
        return;
    }

    // ---- 1. keys.  Protection needs the newest position first: the positions wait in shared memory behind the keys,
    //         or, from EV_STAGE slots per CTA on, are read again
    const bool recent = p.n_recent > 0, staged = p.staged;
    int *pos_s = reinterpret_cast<int *>(keys) + T * p.run;
    int newest = INT_MIN;
    for (int i0 = tid; i0 < n_own; i0 += EV_LOADS * T) {
        float w[EV_LOADS];
        int pos[EV_LOADS];
#pragma unroll
        for (int q = 0; q < EV_LOADS; q++) {
            const int s = s0 + i0 + q * T;
            w[q] = s < s1 ? w_in[s] : 0.0f;
            pos[q] = pos_in && s < s1 ? pos_in[s] : INT_MIN;
        }
#pragma unroll
        for (int q = 0; q < EV_LOADS; q++) {
            const int i = i0 + q * T, s = s0 + i;
            if (i >= n_own) break;
            newest = max(newest, pos[q]);
            keys[i] = pos_in && pos[q] < p.n_first ? KEY_PROTECTED : weight_key(w[q]);
            if (recent && staged) pos_s[i] = pos[q];
            if (s < budget) {
                if (copy_w) w_out[s] = w[q];
                if (copy_pos) pos_out[s] = pos[q];
            }
        }
    }
    if (recent) {
        newest = __reduce_max_sync(0xffffffffu, newest);
        if ((tid & 31) == 0) atomicMax(&sh.max_pos, newest);
        cluster_barrier();
        newest = (int)ld_cluster_u32(cluster_map(&sh.max_pos, (uint32_t)min(tid & 31, C - 1)));
        newest = __reduce_max_sync(0xffffffffu, newest);
    }
    // the first digit's histogram, from the final keys (each thread its own slots')
    const long long recent_from = (long long)newest - p.n_recent;  // positions above are protected
    for (int i0 = tid; i0 < n_own; i0 += EV_LOADS * T) {
        int pos[EV_LOADS];
        if (recent) {
#pragma unroll
            for (int q = 0; q < EV_LOADS; q++) {
                const int i = i0 + q * T;
                pos[q] = i >= n_own ? INT_MIN : staged ? pos_s[i] : pos_in[s0 + i];
            }
        }
#pragma unroll
        for (int q = 0; q < EV_LOADS; q++) {
            const int i = i0 + q * T;
            if (i >= n_own) break;
            uint32_t key = keys[i];
            if (recent && pos[q] > recent_from) keys[i] = key = KEY_PROTECTED;
            atomicAdd(&sh.hist[0][key >> 21], 1u);
        }
    }

    // ---- 2. the budget-th largest key: `prefix` holds its digits found so far, `need` of the keys that share
    //         them are kept
    uint32_t prefix = 0;
    int need = budget, equal = 0;
    uint32_t *close = reinterpret_cast<uint32_t *>(pos_s);  // the keys that share the first digit, as far as they fit
    const int close_cap = staged ? T * p.run : 0;
#pragma unroll
    for (int digit = 0; digit < 3; digit++) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bins = digit == 2 ? 1024 : 2048;
        unsigned *hist = sh.hist[digit];
        if (digit == 1) {
            for (int i = tid; i < n_own; i += T) {
                const uint32_t key = keys[i];
                if (key >> 21 != prefix >> 21) continue;
                atomicAdd(&hist[(key >> 10) & 2047], 1u);
                const int at_close = atomicAdd(&sh.n_close, 1);
                if (at_close < close_cap) close[at_close] = key;
            }
        } else if (digit == 2) {
            const bool listed = sh.n_close <= close_cap;
            const uint32_t *from = listed ? close : keys;
            const int n = listed ? sh.n_close : n_own;
            for (int i = tid; i < n; i += T)
                if (from[i] >> 10 == prefix >> 10) atomicAdd(&hist[from[i] & 1023], 1u);
        }
        cluster_barrier();
        // over the cluster: each CTA adds the others' counts of its share of the bins to its own, four bins of one
        // CTA per thread, and then everyone reads every share
        const int share = bins / C;  // C is a power of two
        if (C > 1) {
            const int r = tid / (share / 4), bin = rank * share + 4 * (tid % (share / 4));
            if (r < C && r != rank) {
                const uint4 x = ld_cluster_u32x4(cluster_map(hist + bin, (uint32_t)r));
                if (x.x) atomicAdd(&hist[bin], x.x);
                if (x.y) atomicAdd(&hist[bin + 1], x.y);
                if (x.z) atomicAdd(&hist[bin + 2], x.z);
                if (x.w) atomicAdd(&hist[bin + 3], x.w);
            }
            cluster_barrier();
        }
        // thread t takes the t-th four bins from the top
        uint4 cnt{0, 0, 0, 0};
        const int bin0 = bins - 4 - 4 * tid;
        if (bin0 >= 0) cnt = ld_cluster_u32x4(cluster_map(hist + bin0, (uint32_t)(bin0 / share)));
        int all, above = block_prefix<T>((int)(cnt.x + cnt.y + cnt.z + cnt.w), sh.warp_tot[digit], &all);
        const int c4[4] = {(int)cnt.w, (int)cnt.z, (int)cnt.y, (int)cnt.x};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (above < need && need <= above + c4[q]) {
                sh.found[digit][0] = bin0 + 3 - q;
                sh.found[digit][1] = above;
                sh.found[digit][2] = c4[q];
            }
            above += c4[q];
        }
        __syncthreads();
        prefix |= (uint32_t)sh.found[digit][0] << shift;
        need -= sh.found[digit][1];
        equal = sh.found[digit][2];
    }

    // ---- 3. holes and movers of this thread's run
    const int r0 = tid * run, r1 = min(n_own, r0 + run);
    int tie_rank = 0;  // of this thread's first key equal to the threshold, over the cluster
    if (equal > need) {
        int ties = 0, all;
        for (int i = r0; i < r1; i++) ties += keys[i] == prefix;
        tie_rank = block_prefix<T>(ties, sh.warp_tot[3], &all);
        if (C > 1) {
            if (tid == 0) sh.ties = all;
            cluster_barrier();
            const int r = tid & 31;
            const int x = r < rank ? (int)ld_cluster_u32(cluster_map(&sh.ties, (uint32_t)r)) : 0;
            tie_rank += __reduce_add_sync(0xffffffffu, x);
        }
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
    // at most 33792 slots per CTA: both counts fit in half an unsigned word
    int both;
    const uint32_t ranks = (uint32_t)block_prefix<T>((int)((uint32_t)__popcll(holes) << 16) | __popcll(movers), sh.warp_tot[4], &both);
    int *list = reinterpret_cast<int *>(keys);  // every key is read: holes from the front, movers from the back
    const int last = T * run - 1;
    for (int j = (int)(ranks >> 16); holes; holes &= holes - 1) list[j++] = s0 + r0 + __ffsll(holes) - 1;
    for (int j = (int)(ranks & 0xFFFFu); movers; movers &= movers - 1) list[last - j++] = s0 + r0 + __ffsll(movers) - 1;
    if (tid == 0) {
        sh.counts[0] = (int)((uint32_t)both >> 16);
        sh.counts[1] = both & 0xFFFF;
    }
    cluster_barrier();
    if (tid < 32) {  // exclusive prefixes over the cluster, lane r for CTA r
        int h = 0, m = 0;
        if (tid < C) {
            h = (int)ld_cluster_u32(cluster_map(&sh.counts[0], (uint32_t)tid));
            m = (int)ld_cluster_u32(cluster_map(&sh.counts[1], (uint32_t)tid));
        }
        int hi = h, mi = m;
#pragma unroll
        for (int o = 1; o < EV_CLUSTER_MAX; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, hi, o), y = __shfl_up_sync(0xffffffffu, mi, o);
            if (tid >= o) {
                hi += x;
                mi += y;
            }
        }
        if (tid < C) {
            sh.pre_h[tid + 1] = hi;
            sh.pre_m[tid + 1] = mi;
        }
        if (tid == 0) sh.pre_h[0] = sh.pre_m[0] = 0;
    }
    __syncthreads();

    // ---- 4. this CTA's share of the moves (holes and movers are equally many; if they should not be, nothing moves)
    if (tid == 0 && sh.pre_m[C] != sh.pre_h[C]) record_error(p.err, DEVERR_BADLEN);
    const long long n_moves = sh.pre_m[C] == sh.pre_h[C] ? sh.pre_m[C] : 0;
    const int m0 = (int)(n_moves * rank / C), m1 = (int)(n_moves * (rank + 1) / C);
    // of them this part's rows
    const int k0 = m0 + (int)((long long)(m1 - m0) * part / parts), k1 = m0 + (int)((long long)(m1 - m0) * (part + 1) / parts);
    const long long head_off = (long long)item * p.item_stride + (long long)kvh * p.max_tokens * (NB * BLOCK_BYTES);
    // up to 32 moves at a time per warp, a lane looking each of them up
    auto slot_of = [&](const int *pre, int j, bool mover) {
        int r = 0;
        while (r + 1 < C && pre[r + 1] <= j) r++;
        return (int)ld_cluster_u32(cluster_map(mover ? &list[last - (j - pre[r])] : &list[j - pre[r]], (uint32_t)r));
    };
    auto move_stats = [&](int src, int dst) {
        w_out[dst] = w_in[src];
        if (pos_in) pos_out[dst] = pos_in[src];
    };
    // few moves are spread over the warps
    const int lane = tid & 31, step = max(1, min(32, (k1 - k0 + (T / 32) - 1) / (T / 32)));
    for (int b = k0 + (tid >> 5) * step; b < k1; b += (T / 32) * step) {
        const int n = min(step, k1 - b);
        int src = 0, dst = 0;
        if (lane < n) {
            src = slot_of(sh.pre_m, b + lane, true);
            dst = slot_of(sh.pre_h, b + lane, false);
            if (part == 0) move_stats(src, dst);
        }
        move_rows<NB>(p.k + head_off, p.v + head_off, src, dst, n);
    }
    // the sums and positions of the other parts' rows: written by the part that copied the rest of them
    if (PARTS && part == 0)
        for (int j = k1 + tid; j < m1; j += T) move_stats(slot_of(sh.pre_m, j, true), slot_of(sh.pre_h, j, false));
    if (C > 1) cluster_barrier();  // no CTA leaves while another reads its list
}

// lens_out[i] = min(len_i, budget) in place: after the eviction has read every length.
__global__ void evict_lens_kernel(const int *lens, int len0, int len_step, int len_cap, int budget, int n, int *out) {
    grid_dependency_wait();
    grid_dependents_launch();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) out[i] = min(min(max(lens ? lens[i] : len0 + i * len_step, 0), len_cap), budget);
}

template <int NB, int T, bool PARTS>
int launch_evict(const EvictParams &p, int cluster, dim3 grid, cudaStream_t stream) {
    size_t smem = (size_t)T * p.run * (p.staged ? 2 : 1) * sizeof(uint32_t);
    // few CTAs: one per SM (two would share an SM while others idle)
    if ((long long)grid.x * grid.y * grid.z <= device_info()->sm_count && smem < EV_ALONE) smem = EV_ALONE;
    // the dynamic shared-memory opt-in is a per-device function attribute
    static std::mutex mu;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return fail_cuda(e, "tqk_evict_q8: cudaGetDevice");
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(evict_kernel<NB, T, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     EV_KEY_BYTES_MAX);
            if (e != cudaSuccess) return fail_cuda(e, "tqk_evict_q8: kernel attributes");
            ready[dev] = true;
        }
    }
    if (cluster == 1) return launch_pdl(evict_kernel<NB, T, PARTS>, grid, dim3(T), smem, stream, p);
    return launch_pdl_cluster(evict_kernel<NB, T, PARTS>, grid, dim3(T), smem, stream, (unsigned)cluster, p);
}

template <int T, bool PARTS>
int dispatch_evict(int nb, const EvictParams &p, int cluster, dim3 grid, cudaStream_t stream) {
    switch (nb) {
        case 1: return launch_evict<1, T, PARTS>(p, cluster, grid, stream);
        case 2: return launch_evict<2, T, PARTS>(p, cluster, grid, stream);
        case 4: return launch_evict<4, T, PARTS>(p, cluster, grid, stream);
        default: return launch_evict<8, T, PARTS>(p, cluster, grid, stream);
    }
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
    if (max_len > 0 || a->lens || a->lens_out) {  // also where max_len is 0: device lengths above it are reported
        EvictParams p{};
        p.k = reinterpret_cast<uint8_t *>(a->k);
        p.v = reinterpret_cast<uint8_t *>(a->v);
        p.item_stride = a->item_stride * BLOCK_BYTES;
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
        // CTAs per (item, head), as far as a cluster goes: as many as hold 8192 slots each (32 layers of 8 heads at 4097
        // rows: 11 us with one, 27 us with two), and down to 1024 each while every CTA has an SM (8 heads, half of
        // 8192 rows evicted: 31 us with one CTA per head, 17 us with eight).  Then also 1024 threads instead of 512,
        // which bring the work per thread down and more moves in flight (8 heads, a quarter of 131072 rows kept: 87 and
        // 69 us); up to 4096 slots they do not pay
        int cluster = 1;
        while (cluster < EV_CLUSTER_MAX && cluster * EV_STAGE < max_len) cluster *= 2;
        const long long units = (long long)a->n_items * a->n_kv_heads;
        while (cluster < EV_CLUSTER_MAX && cluster * EV_NARROW < max_len && 2 * cluster * units <= device_info()->sm_count)
            cluster *= 2;
        // Moving many rows keeps the SMs that do it busy for longer than finding them.  Where SMs are left over and the
        // sums and positions go elsewhere (a cluster may still read them when another is done), several clusters share
        // a head's moves, each finding them for itself.  Half of 131072 rows kept, in place (one cluster per head) and
        // elsewhere (so): 1 head 61 and 33 us, 2 heads 63 and 39 us, 4 heads 65 and 53 us.  Only up to half of the SMs:
        // 16 clusters of 8 do not all run at once (8 heads, at the time 85 us with 8 clusters: 123 us; 8 clusters of 16
        // CTAs do not either: 112 us)
        int parts = 1;
        const long long busy = units * cluster;
        const int moves = a->budget < max_len - a->budget ? a->budget : max_len - a->budget;  // at most, at max_len
        if (cluster == EV_CLUSTER_MAX && moves >= EV_PARTS_MOVES && a->weight_out != a->weight &&
            (!a->position || a->position_out != a->position))
            while (parts < EV_PARTS_MAX && 2 * parts * busy <= device_info()->sm_count / 2) parts *= 2;
        const dim3 grid((unsigned)(cluster * parts), (unsigned)a->n_kv_heads, (unsigned)a->n_items);
        const bool wide = max_len > EV_STAGE / 2 && (long long)grid.x * grid.y * grid.z <= device_info()->sm_count;
        const int threads = wide ? EV_WIDE : EV_THREADS;
        p.run = ((max_len + cluster * threads - 1) / (cluster * threads)) | 1;
        p.staged = max_len <= cluster * EV_STAGE;
        p.lens_out = a->lens_out != a->lens ? a->lens_out : nullptr;
        rc = parts > 1 ? dispatch_evict<EV_WIDE, true>(nb, p, cluster, grid, st)
             : wide    ? dispatch_evict<EV_WIDE, false>(nb, p, cluster, grid, st)
                       : dispatch_evict<EV_THREADS, false>(nb, p, cluster, grid, st);
        if (rc) return rc;
    }
    if (!a->lens_out || a->lens_out != a->lens) return TQK_OK;
    return launch_pdl(evict_lens_kernel, dim3((unsigned)((a->n_items + 255) / 256)), dim3(256), 0, st, a->lens, a->len0,
                      a->len_step, max_len, a->budget, a->n_items, a->lens_out);
}
