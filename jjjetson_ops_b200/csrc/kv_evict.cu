// Eviction from a paged cache by accumulated attention weight: of every sequence and key-value head the first and the last tokens stay and
// of the others those of the largest weight, in their order.  Two launches: one finds the tokens, one moves their keys and values.
//
// Finding: the weight that the last kept token has is found by its bits, 11, 11 and 10 at a time, from histograms (a sort would move every
// weight several times; this reads them once from memory).  The blocks of a cluster share one head: each holds its slice of the weights in
// shared memory throughout, and reads the others' histograms there.  One long sequence has few heads, so this is what brings more than one
// SM to a head.  What bounds it is latency: three histograms one after the other.
//
// Moving: bound by bytes, each kept row read and written once.  Into other pages all rows move at once.  Within the same pages a row may only
// be overwritten after it was read: a block has a column (32 bytes or more) of all rows of a head to itself and takes the rows in their
// order, a tile of loads before the tile's stores (a row never moves back, so later tiles read behind all earlier stores).
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

constexpr int SELECT_THREADS = 1024;
constexpr int SELECT_WARPS = SELECT_THREADS / 32;
constexpr int MAX_CLUSTER = 8;
static_assert(SELECT_WARPS == 32, "a lane for every warp");
constexpr int DIGITS = 3;
constexpr int BINS = 2048;
constexpr int BINS_PER_THREAD = BINS / SELECT_THREADS;
constexpr int64_t MAX_SLICE = 48 * 1024;  // weights of one block

struct EvictArgs {
    KvIndex ix;
    const int32_t *lens;
    const float *weights;
    int64_t weights_stride;
    int32_t *kept, *new_lens;
    float *new_weights;
    int64_t new_weights_stride;
    int kv_heads, max_len, keep, recent, sinks;
    // moving
    KvIndex to;
    char *k, *v;
    int row_bytes;
    int *fault;
};

__device__ __forceinline__ int tokens_of(const EvictArgs &a, int seq) { return min(kv_length(a.ix, a.lens[seq]), a.max_len); }

// Larger weights have larger keys; NaN counts as minus infinity, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

struct Counts {
    int above, equal;
};

// (two blocks on an SM, which leaves 32 registers and spills one: with one block, of 38, 128 blocks in clusters of eight take turns.  A whole
// call into other pages, its data not in L2, us with one / two: 17 x 4 heads of 27173 down to 2000 70.7 / 56.4, down to 8000 142 / 130, 2 x 8 of 20000
// to 4000 48.2 / 42.0, 6 x 8 of 9000 to 2000 48.1 / 42.0, 24 x 8 of 5000 to 1000 58.4 / 56.4; 8 of 100003 to 16000 54.3 both.  21 x 8 of 3000
// to 1000 within their pages lose: 37.9 / 42.0)
__global__ void __launch_bounds__(SELECT_THREADS, 2) evict_select_kernel(const EvictArgs a) {
    extern __shared__ __align__(16) float w[];  // this block's slice
    __shared__ __align__(16) uint32_t bins[DIGITS][BINS];
    __shared__ uint32_t sums[SELECT_WARPS];
    __shared__ uint32_t found_bin, found_left;
    __shared__ Counts warp_counts[SELECT_WARPS], block_counts;
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int parts = cluster.num_blocks(), part = cluster.block_rank();
    const int head = blockIdx.x / parts, seq = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t at = (int64_t)seq * a.kv_heads + head;
    const float *from = a.weights + at * a.weights_stride;
    float *new_w = a.new_weights + at * a.new_weights_stride;
    int32_t *kept = a.kept + at * a.keep;
    const int n = tokens_of(a, seq), stays = min(n, a.keep);
    const int thread = part * SELECT_THREADS + threadIdx.x, threads = parts * SELECT_THREADS;

    for (int behind = a.keep - stays - thread; behind > 0; behind -= threads) kept[a.keep - behind] = -1;  // (a step beyond keep may be beyond 2^31)
    if (n <= a.keep) {  // all stay
        for (int i = thread; i < n; i += threads) {
            kept[i] = i;
            if (new_w != from) new_w[i] = from[i];
        }
        for (int64_t i = n + thread; i < a.max_len; i += threads) new_w[i] = 0.f;
        return;
    }

    const int slice = ((n + parts - 1) / parts + 31) / 32 * 32;
    const int first = min(n, part * slice), mine = min(n, first + slice) - first;
    for (int i = threadIdx.x; i < DIGITS * BINS / 4; i += SELECT_THREADS) reinterpret_cast<uint4 *>(&bins[0][0])[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int low = a.sinks, high = n - a.recent;  // candidates
    const int c0 = max(low - first, 0), c1 = min(high - first, mine);
    uint32_t left = (uint32_t)(a.keep - a.sinks - a.recent), prefix = 0;
    // the slice into shared memory, eight loads of a thread at a time, and into the first histogram
    for (int i0 = threadIdx.x; i0 < mine; i0 += 8 * SELECT_THREADS) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * SELECT_THREADS;
            x[u] = i < mine ? from[first + i] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * SELECT_THREADS;
            if (i < mine) w[i] = x[u];
            if (i >= c0 && i < c1) atomicAdd(&bins[0][key_of(x[u]) >> 21], 1u);
        }
    }

    // the weight of the last token that stays, of those that are not kept anyway
    const auto everybody = [&]() {
        if (parts > 1) cluster.sync();
        else __syncthreads();
    };
    if (left > 0) {
#pragma unroll
        for (int digit = 0; digit < DIGITS; ++digit) {
            if (digit > 0) {
                for (int i = c0 + (int)threadIdx.x; i < c1; i += SELECT_THREADS) {
                    const uint32_t key = key_of(w[i]);
                    if (key >> (digit == 1 ? 21 : 10) == prefix) atomicAdd(&bins[digit][digit == 1 ? key >> 10 & (BINS - 1) : key & 1023u], 1u);
                }
            }
            everybody();
            uint2 sum = make_uint2(0, 0);  // this thread's two bins, over the blocks
#pragma unroll 4
            for (int p = 0; p < parts; ++p) {
                const uint2 x = reinterpret_cast<const uint2 *>(cluster.map_shared_rank(&bins[digit][0], p))[threadIdx.x];
                sum = make_uint2(sum.x + x.x, sum.y + x.y);
            }
            // how many lie in higher bins
            const uint32_t own = sum.x + sum.y;
            uint32_t up = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_down_sync(0xFFFFFFFFu, up, o);
                if (lane + o < 32) up += u;
            }
            if (lane == 0) sums[warp] = up;
            __syncthreads();
            const uint32_t behind = __reduce_add_sync(0xFFFFFFFFu, lane > warp ? sums[lane] : 0u);
            uint32_t above = up - own + behind;
            if (above < left && left <= above + own) {
                const bool upper = left <= above + sum.y;
                found_bin = BINS_PER_THREAD * threadIdx.x + (upper ? 1 : 0);
                found_left = left - above - (upper ? 0 : sum.y);
            }
            __syncthreads();
            left = found_left;
            prefix = prefix << (digit == 2 ? 10 : 11) | found_bin;
        }
    } else {
        prefix = 0xFFFFFFFFu;  // above every key
        everybody();           // all slices are loaded before weights are written
    }
    const uint32_t last_key = prefix;
    const int of_equal = (int)left;  // so many of those with the last weight stay, the first ones

    // places: every warp has a span of the slice
    const int span = (mine + 32 * SELECT_WARPS - 1) / (32 * SELECT_WARPS) * 32;
    const int s0 = min(mine, warp * span), s1 = min(mine, s0 + span);
    const auto flags = [&](int i, bool *above, bool *equal) {
        const bool in = i < s1, candidate = in && i >= c0 && i < c1;
        const uint32_t key = in ? key_of(w[i]) : 0;
        *above = in && (!candidate || key > last_key);
        *equal = candidate && key == last_key;
    };
    Counts count = {0, 0};
    for (int i = s0 + lane; i - lane < s1; i += 32) {
        bool above, equal;
        flags(i, &above, &equal);
        count.above += __popc(__ballot_sync(0xFFFFFFFFu, above));
        count.equal += __popc(__ballot_sync(0xFFFFFFFFu, equal));
    }
    if (lane == 0) warp_counts[warp] = count;
    __syncthreads();
    const Counts of_lane = warp_counts[lane];
    if (parts > 1) {
        if (warp == 0) {
            const Counts all = {__reduce_add_sync(0xFFFFFFFFu, of_lane.above), __reduce_add_sync(0xFFFFFFFFu, of_lane.equal)};
            if (lane == 0) block_counts = all;
        }
        cluster.sync();
    }
    Counts before = {__reduce_add_sync(0xFFFFFFFFu, lane < warp ? of_lane.above : 0), __reduce_add_sync(0xFFFFFFFFu, lane < warp ? of_lane.equal : 0)};
    if (part > 0) {
        Counts c = {0, 0};
        if (lane < part) c = *cluster.map_shared_rank(&block_counts, lane);
        before.above += __reduce_add_sync(0xFFFFFFFFu, c.above), before.equal += __reduce_add_sync(0xFFFFFFFFu, c.equal);
    }
    for (int i = s0 + lane; i - lane < s1; i += 32) {
        bool above, equal;
        flags(i, &above, &equal);
        const uint32_t higher = __ballot_sync(0xFFFFFFFFu, above), same = __ballot_sync(0xFFFFFFFFu, equal);
        const uint32_t lower_lanes = (1u << lane) - 1;
        const int rank = before.equal + __popc(same & lower_lanes);
        if (above || (equal && rank < of_equal)) {
            const int to = before.above + __popc(higher & lower_lanes) + min(rank, of_equal);
            kept[to] = first + i;
            new_w[to] = w[i];
        }
        before.above += __popc(higher);
        before.equal += __popc(same);
    }
    for (int64_t i = stays + thread; i < a.max_len; i += threads) new_w[i] = 0.f;
    if (parts > 1) cluster.sync();  // no block ends while another reads its counts
}

__device__ __forceinline__ int64_t place_of(const KvIndex &ix, int seq, int token, int *fault) {
    const int64_t to = kv_offset(ix, (uint32_t)token, ix.table[(int64_t)seq * ix.table_stride + kv_page_of(ix, (uint32_t)token)]);
    if (to < 0) report_bad_page(fault);
    return to;
}
// (the list of kept tokens says where a sequence ends, so that new_lens may be lens)
__device__ __forceinline__ void write_length(const EvictArgs &a, int seq) { a.new_lens[seq] = min(tokens_of(a, seq), a.keep); }

constexpr int MOVE_THREADS = 256;
constexpr int MOVE_AT_ONCE = 4;  // rows per thread

// 2^shift threads per row of 16-byte chunks (a row has row_bytes / 16 of them).
template <typename E>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const EvictArgs a, int shift) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int head = blockIdx.y, seq = blockIdx.z;
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) write_length(a, seq);
    const int32_t *kept = a.kept + ((int64_t)seq * a.kv_heads + head) * a.keep;
    const int chunk = threadIdx.x & ((1 << shift) - 1), rows = MOVE_THREADS >> shift;
    const bool inside = chunk * 16 < a.row_bytes;
    const int64_t column = (int64_t)head * a.ix.stride_head * (int)sizeof(E) + chunk * 16;
    const uint32_t j0 = blockIdx.x * (uint32_t)(rows * MOVE_AT_ONCE) + (threadIdx.x >> shift);  // (the last block's may be above 2^31)
    uint4 k[MOVE_AT_ONCE], v[MOVE_AT_ONCE];
    int64_t to[MOVE_AT_ONCE];
#pragma unroll
    for (int u = 0; u < MOVE_AT_ONCE; ++u) {
        const uint32_t j = j0 + u * rows;
        to[u] = -1;
        if (j >= (uint32_t)a.keep || !inside) continue;
        const int i = kept[j];
        if (i < 0) continue;
        const int64_t from = place_of(a.ix, seq, i, a.fault), there = place_of(a.to, seq, (int)j, a.fault);
        if (from < 0 || there < 0) continue;
        to[u] = there * (int)sizeof(E) + column;
        k[u] = __ldcs(reinterpret_cast<const uint4 *>(a.k + from * (int)sizeof(E) + column));
        v[u] = __ldcs(reinterpret_cast<const uint4 *>(a.v + from * (int)sizeof(E) + column));
    }
#pragma unroll
    for (int u = 0; u < MOVE_AT_ONCE; ++u) {
        if (to[u] < 0) continue;
        *reinterpret_cast<uint4 *>(a.k + to[u]) = k[u];
        *reinterpret_cast<uint4 *>(a.v + to[u]) = v[u];
    }
}

constexpr int SHIFT_THREADS = 512;

// Within the same pages: 2^shift threads have 16 bytes of a row each.
template <typename E>
__global__ void __launch_bounds__(SHIFT_THREADS) evict_shift_kernel(const EvictArgs a, int shift) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int wide = 16 << shift, columns = (a.row_bytes + wide - 1) / wide;
    const int head = blockIdx.y, seq = blockIdx.z;
    const bool values = (int)blockIdx.x >= columns;
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) write_length(a, seq);
    char *rows = values ? a.v : a.k;
    const int chunk = ((int)blockIdx.x - (values ? columns : 0)) * wide + (threadIdx.x & ((1 << shift) - 1)) * 16;
    const bool inside = chunk < a.row_bytes;
    const int64_t column = (int64_t)head * a.ix.stride_head * (int)sizeof(E) + chunk;
    const int32_t *kept = a.kept + ((int64_t)seq * a.kv_heads + head) * a.keep;
    // Indices ascend: if the last of them is in its place, all are.  (Should another block have written the new length already, in the place
    // of the old one, this is the same number.)
    const int stays = min(tokens_of(a, seq), a.keep);
    if (stays == 0 || kept[stays - 1] == stays - 1) return;
    const int rows_at_once = SHIFT_THREADS >> shift;
    for (int j0 = 0; j0 < stays; j0 += rows_at_once * MOVE_AT_ONCE) {
        uint4 x[MOVE_AT_ONCE];
        int64_t to[MOVE_AT_ONCE];
#pragma unroll
        for (int u = 0; u < MOVE_AT_ONCE; ++u) {
            const int j = j0 + u * rows_at_once + (int)(threadIdx.x >> shift);
            to[u] = -1;
            if (j >= a.keep || !inside) continue;
            const int i = kept[j];
            if (i < 0 || i == j) continue;
            const int64_t from = place_of(a.ix, seq, i, a.fault), there = place_of(a.ix, seq, j, a.fault);
            if (from < 0 || there < 0) continue;
            to[u] = there * (int)sizeof(E) + column;
            x[u] = *reinterpret_cast<const uint4 *>(rows + from * (int)sizeof(E) + column);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < MOVE_AT_ONCE; ++u) {
            if (to[u] >= 0) *reinterpret_cast<uint4 *>(rows + to[u]) = x[u];
        }
    }
}

template <typename... A>
int launch(cudaStream_t st, void (*kernel)(A...), dim3 grid, int threads, size_t smem, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    return JQ_OK;
}

template <typename E>
int launch_move(cudaStream_t st, const EvictArgs &a, int64_t seqs, bool in_place) {
    if (in_place) {
        // columns as wide as leave all rows in one tile, 32 bytes at least: 1024 rows of 256 bytes in columns of 64 11.8 us, of 32 8.2
        int shift = 1;
        while ((16 << shift) < a.row_bytes && ((SHIFT_THREADS * MOVE_AT_ONCE) >> (shift + 1)) >= a.keep) ++shift;
        const int columns = (a.row_bytes + (16 << shift) - 1) / (16 << shift);
        return launch(st, evict_shift_kernel<E>, dim3((unsigned)(2 * columns), (unsigned)a.kv_heads, (unsigned)seqs), SHIFT_THREADS, 0, 0, a, shift);
    }
    int shift = 0;
    while (16 << shift < a.row_bytes) ++shift;
    const int64_t rows = (MOVE_THREADS >> shift) * MOVE_AT_ONCE;
    return launch(st, evict_move_kernel<E>, dim3((unsigned)((a.keep + rows - 1) / rows), (unsigned)a.kv_heads, (unsigned)seqs), MOVE_THREADS, 0, 0, a, shift);
}

}  // namespace

}  // namespace jq

using namespace jq;

extern "C" {

int64_t jq_kv_evict_max_len(void) { return MAX_CLUSTER * MAX_SLICE; }

int jq_kv_evict_device(void *stream, const jq_kv_cache *cache, const int32_t *d_lens, const float *d_weights, int64_t weights_stride,
                       int64_t max_len, int64_t keep, int64_t recent, int64_t sinks, const int32_t *d_new_page_table,
                       int64_t new_max_pages, int64_t new_table_stride, int32_t *d_kept, int32_t *d_new_lens,
                       float *d_new_weights, int64_t new_weights_stride) {
    EvictArgs a = {};
    if (int rc = check_kv_cache(cache, &a.ix)) return rc;
    if (max_len < 0 || keep <= 0 || recent < 0 || sinks < 0)
        return set_error(JQ_ERR_INVALID_ARG, "evict: a size is negative, or nothing is to be kept");
    if (recent > keep || sinks > keep - recent)
        return set_error(JQ_ERR_INVALID_ARG, "evict: sinks = %lld and recent = %lld are more than keep = %lld", (long long)sinks, (long long)recent, (long long)keep);
    if (max_len > jq_kv_evict_max_len())
        return set_error(JQ_ERR_TOO_LARGE, "evict: max_len = %lld is above %lld", (long long)max_len, (long long)jq_kv_evict_max_len());
    if (keep > 0x7FFFFF00 || cache->num_seqs > 65535) return set_error(JQ_ERR_TOO_LARGE, "evict: keep, or more than 65535 sequences");
    if (weights_stride < max_len || new_weights_stride < max_len)
        return set_error(JQ_ERR_INVALID_ARG, "evict: rows of the weights overlap");
    if (cache->num_seqs == 0) return JQ_OK;
    if (d_lens == nullptr || d_kept == nullptr || d_new_lens == nullptr || (max_len > 0 && (d_weights == nullptr || d_new_weights == nullptr)))
        return set_error(JQ_ERR_INVALID_ARG, "evict: null pointer");
    if ((((uintptr_t)d_lens | (uintptr_t)d_weights | (uintptr_t)d_new_page_table | (uintptr_t)d_kept | (uintptr_t)d_new_lens | (uintptr_t)d_new_weights) & 3u) != 0)
        return set_error(JQ_ERR_ALIGN, "evict: tables, lengths and weights must be 4-byte aligned");
    if (d_new_weights == d_weights && new_weights_stride != weights_stride)
        return set_error(JQ_ERR_INVALID_ARG, "evict: weights in place have one stride");
    const bool in_place = d_new_page_table == nullptr;
    a.to = a.ix;
    if (!in_place) {
        if (d_new_page_table == cache->d_page_table)  // rows would be overwritten before they are read
            return set_error(JQ_ERR_INVALID_ARG, "evict: the new page table is the cache's own; without one tokens stay within their pages");
        if (new_max_pages < 0 || new_max_pages > 0x7FFFFFFF || (keep + cache->page_size - 1) / cache->page_size > new_max_pages)
            return set_error(JQ_ERR_INVALID_ARG, "evict: %lld new pages do not hold %lld tokens", (long long)new_max_pages, (long long)keep);
        if (new_table_stride < new_max_pages && cache->num_seqs > 1)
            return set_error(JQ_ERR_INVALID_ARG, "evict: rows of the new page table overlap");
        a.to.table = d_new_page_table;
        a.to.table_stride = new_table_stride;
        a.to.max_pages = (int32_t)new_max_pages;
    }
    a.lens = d_lens, a.weights = d_weights, a.weights_stride = weights_stride;
    a.kept = d_kept, a.new_lens = d_new_lens, a.new_weights = d_new_weights, a.new_weights_stride = new_weights_stride;
    a.kv_heads = (int)cache->num_kv_heads, a.max_len = (int)max_len, a.keep = (int)keep, a.recent = (int)recent, a.sinks = (int)sinks;
    a.k = static_cast<char *>(cache->d_k), a.v = static_cast<char *>(cache->d_v);
    a.row_bytes = (int)cache->head_dim * kv_element_bytes(cache->type);
    a.fault = device_fault_ptr();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Blocks per head: one for every 2048 weights, but no more than two for an SM, and as many as it takes for a slice to fit (two slices of up to
    // some 22 000 weights fit on an SM; blocks with longer ones wait for one another where there are more than SMs)
    DeviceCaps caps;
    if (int rc = device_caps(&caps)) return rc;
    const int64_t heads = a.kv_heads * cache->num_seqs;
    int parts = 1;
    while (parts < MAX_CLUSTER && max_len > 2048 * parts && (2 * parts * heads <= 2 * caps.sm_count || max_len > MAX_SLICE * parts)) parts *= 2;
    const size_t smem = sizeof(float) * (size_t)(((max_len + parts - 1) / parts + 31) / 32 * 32);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(evict_select_kernel), (int)(smem > 32 * 1024 ? sizeof(float) * MAX_SLICE : 32 * 1024))) return rc;
    if (int rc = launch(st, evict_select_kernel, dim3((unsigned)(a.kv_heads * parts), (unsigned)cache->num_seqs), SELECT_THREADS, smem, parts, a)) return rc;
    if (cache->type == JQ_KV_E4M3) return launch_move<uint8_t>(st, a, cache->num_seqs, in_place);
    return launch_move<uint16_t>(st, a, cache->num_seqs, in_place);
}

}  // extern "C"
