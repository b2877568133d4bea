// Attention of one query token per row over a paged cache: out = sum_i p_i v_i, p = softmax(scale q . k_i).
//
// One pass over keys and values with the running maximum and sum of the softmax, in base 2: with m the largest logit so far,
//   l <- l 2^(m - m') + sum 2^(s_i - m'),   o <- o 2^(m - m') + sum 2^(s_i - m') v_i.
//
// What bounds it: the bytes of the cache, each read once for all query heads that share it.  The products run on the tensor cores all the
// same: with eight query heads to a key head an fp32 multiply-add per head and element would take as long as the bytes.  Keys are the
// rows of the first product (16 keys x 8 heads), values, transposed on their way out of shared memory, those of the second
// (16 elements x 8 heads), so the heads are the narrow side and few heads waste little (mma.sync: 8 columns are half of the narrowest
// tcgen05 tile, and a warp that needs no other one keeps its data in registers between the two products).
// Queries and probabilities are fp32 and are multiplied as the sum of two fp16 or three bf16 numbers (22 and 24 bits), whose products
// with a 16-bit element are exact; so nothing is rounded to fewer than 22 bits, and the sums are fp32.
//
// The work is cut into units of 16 keys of one row and key head, all units of the call laid end to end, and every block takes an equal
// stretch: long and short rows need no plan on the host, and lengths stay on the device.  The warps of a block take its units in turn, each
// with a ring of stages of its own (asynchronous 16-byte copies) that runs on across the ends of rows.  Where a block's stretch holds all
// of a row's key head it writes the output, else its part; the block that finds itself the last of a row's adds the parts, in
// their order, so the result does not depend on who came last.
#include "kv_cache.cuh"

#include <cmath>

namespace jq {

namespace {

constexpr int UNIT = 16;          // keys
constexpr int RING_BYTES = 192 * 1024;
constexpr int MAX_BLOCKS = 256;   // parts that the last block can weigh in its shared memory

struct AttnArgs {
    const float *q;
    int64_t q_row, q_head;
    const char *k, *v;
    KvIndex ix;
    const int32_t *lens, *seqs;
    float *out;
    uint8_t *xq;
    float scale_log2;  // scale * k_scale / ln 2
    float v_scale;
    int rows, q_heads, kv_heads, group, dim, window;
    int tiles;         // parts of a group that are computed apart (groups of more heads than one pass takes)
    int n_super, order, s_mode;
    // workspace
    int *counters;
    float *parts;
    float2 *norms;     // [rows][q_heads]: largest logit, 1 / sum (with weights)
    float *logits;     // [rows][kv_heads][positions][group] (with weights)
    int64_t positions;
    int *fault;
};

// ---- element types: how 16 keys x 16 elements become operands ---------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {
    const int n = there ? 16 : 0;  // what is not there is filled with zeros, and not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}

template <typename T>
struct Parts;  // how an fp32 pair is split into operands whose sum it is
template <>
struct Parts<KvF16> {
    static constexpr int N = 2;
    static constexpr float UP = 16384.f;  // probabilities are held times 2^14: of a million keys as small as 2^-36 nothing is lost
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&w)[N]) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
        w[0] = *reinterpret_cast<const uint32_t *>(&h);
        w[1] = *reinterpret_cast<const uint32_t *>(&l);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) { mma_f16(d, a, b); }
};
template <>
struct Parts<KvE4m3> : Parts<KvF16> {};  // e4m3 elements become fp16, exactly
template <>
struct Parts<KvBf16> {
    static constexpr int N = 3;
    static constexpr float UP = 1.f;
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&w)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            const float2 f = __bfloat1622float2(h);
            a -= f.x, b -= f.y;
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) { mma_bf16(d, a, b); }
};

__device__ __forceinline__ uint32_t half2_of_e4m3(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return (uint32_t)h.x | (uint32_t)h.y << 16;
}

// Shapes of one instance.
template <typename T, int DP_, int NT_>
struct Shape {
    static constexpr int DP = DP_;                  // head_dim, padded
    static constexpr int NT = NT_;                  // tiles of eight heads
    static constexpr int HEADS = 8 * NT;
    static constexpr int WARPS = DP == 256 ? 4 : 8; // a warp's accumulators and queries are its registers' larger part
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ROW = DP * (int)sizeof(typename T::Element);  // bytes
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int TILE = UNIT * ROW;         // keys, or values, of a unit
    static constexpr int STAGES = RING_BYTES / (WARPS * 2 * TILE);
    static constexpr int RED = NT == 1 ? WARPS : WARPS / 2;  // warps whose results lie in shared memory at a time
    static constexpr int PITCH = DP + 4;            // floats; eight rows' eight elements then lie in different banks
    static constexpr int RING = WARPS * STAGES * 2 * TILE;
    static constexpr int RED_BYTES = RED * HEADS * PITCH * 4;
    static constexpr int STATS = WARPS * HEADS * 8;
    static constexpr int SMEM = RING + RED_BYTES + STATS + WARPS * STAGES * 4;
    static constexpr int PART = HEADS * DP + 2 * HEADS;  // floats of a part: sums, then largest logits, then sums of weights
    static_assert(STAGES >= 3, "a ring of three stages at least");
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(RED_BYTES >= MAX_BLOCKS * HEADS * 4, "the parts' factors take the place of the warps' results");
};

// 16-byte chunk `c` of row `r` of a tile: spread so that eight rows' same chunk lies in different banks.
template <int CHUNKS>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    const int x = CHUNKS >= 8 ? (r & 7) : ((r >> 1) & (CHUNKS - 1));
    return (uint32_t)((r * CHUNKS + (c ^ x)) * 16);
}

// What a row sees.
struct Row {
    int32_t seq, first, end;  // keys [first, end); seq < 0: padding
    int units, unit0;
};
__device__ __forceinline__ Row row_of(const AttnArgs &a, int row) {
    Row r;
    r.seq = a.seqs != nullptr ? a.seqs[row] : row;
    if ((uint32_t)r.seq >= (uint32_t)a.ix.num_seqs) r.seq = -1;
    r.end = r.seq < 0 ? 0 : kv_length(a.ix, a.lens[row]);
    r.first = a.window > 0 && r.end > a.window ? r.end - a.window : 0;
    r.unit0 = r.first / UNIT;
    r.units = r.end > 0 ? (r.end + UNIT - 1) / UNIT - r.unit0 : 0;
    return r;
}

// Inclusive sum over the block; `partial`: one value per warp.  Every thread of the block calls it.
template <int WARPS>
__device__ __forceinline__ int64_t block_inclusive(int64_t v, int64_t *partial, int64_t *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) partial[warp] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += partial[w];
        all += partial[w];
    }
    *total = all;
    return v + before;
}

// Four consecutive elements of the output: element `e` of the heads of one key head's tile (their elements lie end to end), as
// fp32 and as Q8_1.  Every lane of the warp calls it, with consecutive e; `there`: it has elements.
__device__ __forceinline__ void write_output(const AttnArgs &a, int row, int head0, int e, float4 v, bool there) {
    const int64_t n = (int64_t)head0 * a.dim + e;  // within the row
    if (a.out != nullptr && there) *reinterpret_cast<float4 *>(a.out + (int64_t)row * a.q_heads * a.dim + n) = v;
    if (a.xq != nullptr) {
        if (!there) v = make_float4(0.f, 0.f, 0.f, 0.f);
        uint32_t ds;
        const uint32_t q = quantize_group_q8_1(v, a.s_mode, &ds);
        if (there) {
            uint8_t *block = a.xq + q8_block_index(n / SUPER, row, a.n_super, a.rows, a.order) * Q8_BYTES;
            const int i = (int)(n % SUPER);
            *reinterpret_cast<uint32_t *>(block + Q8_QS_OFFSET + i) = q;
            if (i % QK == 0) *reinterpret_cast<uint32_t *>(block + i / QK * 4) = ds;
        }
    }
}

__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }  // a row whose pages are all bad gives zeros

template <typename T, int DP, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(Shape<T, DP, NT>::THREADS, 1) paged_attention_kernel(const AttnArgs a) {
    using S = Shape<T, DP, NT>;
    using P = Parts<T>;
    constexpr bool E4M3 = sizeof(typename T::Element) == 1;
    constexpr int W = S::WARPS;
    extern __shared__ __align__(128) unsigned char smem[];
    float *red = reinterpret_cast<float *>(smem + S::RING);
    float2 *stats = reinterpret_cast<float2 *>(smem + S::RING + S::RED_BYTES);  // [warp][head]: largest logit, sum
    uint32_t *masks = reinterpret_cast<uint32_t *>(smem + S::RING + S::RED_BYTES + S::STATS);
    __shared__ int64_t partial[W];
    __shared__ int start_row;
    __shared__ int64_t start_unit;
    __shared__ int is_last;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int segments_row = a.kv_heads * a.tiles;  // a row's key heads, or tiles of their query heads: each has the row's units

    // ---- the block's stretch ----
    int64_t total = 0;
    for (int r0 = 0; r0 < a.rows; r0 += S::THREADS) {
        const int r = r0 + threadIdx.x;
        int64_t all;
        (void)block_inclusive<W>(r < a.rows ? (int64_t)row_of(a, r).units * segments_row : 0, partial, &all);
        total += all;
    }
    int64_t per_block = (total + gridDim.x - 1) / gridDim.x;
    if (per_block < W) per_block = W;  // a unit for every warp: fewer parts to add
    const int64_t u0 = blockIdx.x * per_block, u1 = min(total, u0 + per_block);
    // rows that see nothing get their zeros here
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const Row x = row_of(a, r);
        if (x.seq < 0 || x.units > 0) continue;
        const int n4 = a.q_heads * a.dim / 4;
        for (int e = threadIdx.x; e < (n4 + 31) / 32 * 32; e += S::THREADS)
            write_output(a, r, 0, 4 * e, make_float4(0.f, 0.f, 0.f, 0.f), e < n4);
    }
    if (u0 >= u1) return;
    {
        int64_t before = 0;
        for (int r0 = 0; r0 < a.rows; r0 += S::THREADS) {
            const int r = r0 + threadIdx.x;
            const int64_t n = r < a.rows ? (int64_t)row_of(a, r).units * segments_row : 0;
            int64_t all;
            const int64_t end = before + block_inclusive<W>(n, partial, &all);
            if (end - n <= u0 && u0 < end) start_row = r, start_unit = u0 - (end - n);
            before += all;
            if (before > u0) break;
        }
        __syncthreads();
    }
    const int count = (int)(u1 - u0);  // units of this block; the host has bounded it

    // ---- the ring: every lane knows where one key of the unit that is copied next lies ----
    const uint32_t ring = smem_u32(smem) + warp * S::STAGES * 2 * S::TILE;
    uint32_t *mask_ring = masks + warp * S::STAGES;
    struct {
        Row row;
        int r, segment, unit;  // unit within the row's
        int left;
        int64_t offset;        // bytes, of this lane's key (lanes 0 to 15)
        bool there;
    } next;
    next.r = start_row;
    next.row = row_of(a, next.r);
    next.segment = (int)(start_unit / next.row.units);
    next.unit = (int)(start_unit - (int64_t)next.segment * next.row.units);
    next.left = count > warp ? (count - warp + W - 1) / W : 0;
    const auto advance = [&](int n) {
        next.unit += n;
        while (next.unit >= next.row.units) {
            next.unit -= next.row.units;
            if (++next.segment == segments_row) {
                next.segment = 0;
                do {
                    next.row = row_of(a, ++next.r);
                } while (next.row.units == 0);
            }
        }
    };
    const auto locate = [&]() {  // asks the page table for the unit after the one that is being copied
        const int key = (next.row.unit0 + next.unit) * UNIT + lane;
        next.there = false;
        next.offset = 0;
        if (lane < UNIT && key >= next.row.first && key < next.row.end) {
            const int64_t to = kv_offset(a.ix, (uint32_t)key, a.ix.table[(int64_t)next.row.seq * a.ix.table_stride + kv_page_of(a.ix, (uint32_t)key)]);
            next.there = to >= 0;
            if (to < 0) report_bad_page(a.fault);
            else next.offset = (to + (int64_t)(next.segment / a.tiles) * a.ix.stride_head) * (int)sizeof(typename T::Element);
        }
    };
    const auto copy = [&](int stage) {
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, next.there);
        if (lane == 0) mask_ring[stage] = mask;
        const uint32_t to = ring + stage * 2 * S::TILE;
        const int c = lane % S::CHUNKS;
        const bool inside = c * 16 < a.dim * (int)sizeof(typename T::Element);
        constexpr int AT_ONCE = 32 / S::CHUNKS;
#pragma unroll
        for (int i = 0; i < UNIT / AT_ONCE; ++i) {
            const int r = lane / S::CHUNKS + i * AT_ONCE;
            const int64_t offset = __shfl_sync(0xFFFFFFFFu, next.offset, r);
            const bool there = inside && (mask >> r & 1u);
            const int64_t at = there ? offset + c * 16 : 0;
            copy16(to + chunk_at<S::CHUNKS>(r, c), a.k + at, there);
            copy16(to + S::TILE + chunk_at<S::CHUNKS>(r, c), a.v + at, there);
        }
    };
    const auto copy_next = [&](int stage) {
        if (next.left > 0) {
            copy(stage);
            if (--next.left > 0) {
                advance(W);
                locate();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (next.left > 0) {
        if (warp > 0) advance(warp);
        locate();
    }
#pragma unroll 1
    for (int s = 0; s < S::STAGES - 1; ++s) copy_next(s);
    int stage = 0;

    // ---- the block's pieces of rows ----
    int row = start_row, done = 0;
    Row seen = row_of(a, row);
    int segment = (int)(start_unit / seen.units);
    int unit = (int)(start_unit - (int64_t)segment * seen.units);
#pragma unroll 1
    while (done < count) {
        const int piece = min(count - done, seen.units - unit);
        const int kv_head = segment / a.tiles, tile = segment - kv_head * a.tiles;
        const int head0 = kv_head * a.group + tile * S::HEADS, heads = min(S::HEADS, a.group - tile * S::HEADS);

        // queries: two or three operands per 16 elements, scaled by a power of two so that fp16 holds them
        uint32_t q[NT][DP / 16][P::N][2];
        float unscale[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int h = 8 * t + (lane >> 2);
            const float *from = a.q + (int64_t)row * a.q_row + (int64_t)(head0 + h) * a.q_head;
            float x[DP / 16][4];
            float largest = 0.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const bool there = h < heads && 16 * s < a.dim;
                // the elements that go with the keys' operands: 2i, 2i + 1, 2i + 8, 2i + 9 of 16, or with e4m3 the four from 4i on
                const int i = lane & 3;
                if (E4M3) {
                    const float4 v = there ? *reinterpret_cast<const float4 *>(from + 16 * s + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[s][0] = v.x, x[s][1] = v.y, x[s][2] = v.z, x[s][3] = v.w;
                } else {
                    const float2 v = there ? *reinterpret_cast<const float2 *>(from + 16 * s + 2 * i) : make_float2(0.f, 0.f);
                    const float2 u = there ? *reinterpret_cast<const float2 *>(from + 16 * s + 2 * i + 8) : make_float2(0.f, 0.f);
                    x[s][0] = v.x, x[s][1] = v.y, x[s][2] = u.x, x[s][3] = u.y;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) largest = fmaxf(largest, fabsf(x[s][j]));
            }
            largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 2));
            // 2^-e with 2^e <= largest, within 2^-100 .. 2^100
            int e = (int)(__float_as_uint(largest) >> 23) - 127;
            e = P::N == 3 || largest == 0.f ? 0 : max(-100, min(100, e));
            const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale_log2;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                uint32_t w0[P::N], w1[P::N];
                P::split(x[s][0] * down, x[s][1] * down, w0);
                P::split(x[s][2] * down, x[s][3] * down, w1);
#pragma unroll
                for (int j = 0; j < P::N; ++j) q[t][s][j][0] = w0[j], q[t][s][j][1] = w1[j];
            }
            // the products' columns: this lane has heads 2i and 2i + 1
            unscale[t][0] = __shfl_sync(0xFFFFFFFFu, up, 8 * (lane & 3));
            unscale[t][1] = __shfl_sync(0xFFFFFFFFu, up, 8 * (lane & 3) + 4);
        }

        float o[NT][DP / 16][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t][s][j] = 0.f;
        }

        int mine = (warp - done % W + W) % W;  // this warp's first unit of the piece
#pragma unroll 1
        for (; mine < piece; mine += W) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
            __syncwarp();
            const uint32_t kt = ring + stage * 2 * S::TILE, vt = kt + S::TILE;
            const uint32_t mask = mask_ring[stage];
            // the stage that was read in the step before this one takes the next unit
            copy_next(stage == 0 ? S::STAGES - 1 : stage - 1);

            // logits of 16 keys x 8 NT heads; four sums, so that no product waits for all the others
            float s4[NT][4][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s4[t][i][j] = 0.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                uint32_t k[4];
                if constexpr (E4M3) {
                    if (s & 1) continue;
                    uint32_t r[4];
                    ldmatrix4(r, kt + chunk_at<S::CHUNKS>(lane & 15, s + (lane >> 4)));
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t k8[4] = {half2_of_e4m3(r[2 * u] & 0xFFFFu), half2_of_e4m3(r[2 * u + 1] & 0xFFFFu),
                                                half2_of_e4m3(r[2 * u] >> 16), half2_of_e4m3(r[2 * u + 1] >> 16)};
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < P::N; ++j) P::mma(s4[t][(2 * u + j) & 3], k8, q[t][s + u][j]);
                    }
                } else {
                    ldmatrix4(k, kt + chunk_at<S::CHUNKS>(lane & 15, 2 * s + (lane >> 4)));
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < P::N; ++j) P::mma(s4[t][(P::N * s + j) & 3], k, q[t][s][j]);
                }
            }

            const bool v0 = mask >> (lane >> 2) & 1u, v1 = mask >> ((lane >> 2) + 8) & 1u;
            uint32_t p[NT][P::N][2];
            float shrink[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float sum = (s4[t][0][j] + s4[t][1][j]) + (s4[t][2][j] + s4[t][3][j]);
                    x[j] = (j < 2 ? v0 : v1) ? sum * unscale[t][j & 1] : -INFINITY;
                }
                if (WEIGHTS) {
                    const int64_t key = (int64_t)(seen.unit0 + unit + mine) * UNIT + (lane >> 2);
                    const int64_t base = ((int64_t)row * a.kv_heads + kv_head) * a.positions;
                    const int h = tile * S::HEADS + 8 * t + 2 * (lane & 3);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool in = key + 8 * (j >> 1) >= seen.first && key + 8 * (j >> 1) < seen.end;
                        if (in && h + (j & 1) < a.group) a.logits[(base + key + 8 * (j >> 1)) * a.group + h + (j & 1)] = x[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(x[j], x[j + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                    top = fmaxf(top, m[t][j]);
                    const float from = top == -INFINITY ? 0.f : top;  // keys of bad pages only, so far
                    shrink[t][j] = exp2f(m[t][j] - from);
                    m[t][j] = top;
                    x[j] = exp2f(x[j] - from) * P::UP;
                    x[j + 2] = exp2f(x[j + 2] - from) * P::UP;
                    l[t][j] = l[t][j] * shrink[t][j] + (x[j] + x[j + 2]);
                }
                uint32_t w0[P::N], w1[P::N];
                P::split(x[0], x[1], w0);
                P::split(x[2], x[3], w1);
#pragma unroll
                for (int j = 0; j < P::N; ++j) p[t][j][0] = transposed(w0[j]), p[t][j][1] = transposed(w1[j]);
            }

            // the tensor cores cut a sum's last bits off instead of rounding: they add up one unit, the sum over units is rounded
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                uint32_t v[4];
                if constexpr (E4M3) {
                    if (s & 1) continue;
                    uint32_t r[4];
                    ldmatrix4_trans(r, vt + chunk_at<S::CHUNKS>((lane & 7) + ((lane >> 4) << 3), s + ((lane >> 3) & 1)));
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        // rows of the product: elements 2i, then 2i + 1, of the 16
                        const uint32_t a0 = __byte_perm(r[u], 0, 0x3120), a1 = __byte_perm(r[u + 2], 0, 0x3120);
                        const uint32_t v8[4] = {half2_of_e4m3(a0 & 0xFFFFu), half2_of_e4m3(a0 >> 16), half2_of_e4m3(a1 & 0xFFFFu), half2_of_e4m3(a1 >> 16)};
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int j = P::N - 1; j >= 0; --j) P::mma(d, v8, p[t][j]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[t][s + u][j] = o[t][s + u][j] * shrink[t][j & 1] + d[j];
                        }
                    }
                } else {
                    ldmatrix4_trans(v, vt + chunk_at<S::CHUNKS>((lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1)));
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = P::N - 1; j >= 0; --j) P::mma(d, v, p[t][j]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[t][s][j] = o[t][s][j] * shrink[t][j & 1] + d[j];
                    }
                }
            }
            if (++stage == S::STAGES) stage = 0;
        }

        // ---- the warps' results to one ----
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 4);
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 8);
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 16);
                if (lane < 4) stats[warp * S::HEADS + 8 * t + 2 * lane + j] = make_float2(m[t][j], l[t][j]);
            }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w * S::HEADS + 8 * t + 2 * (lane & 3) + j].x);
                const float f = exp2f(m[t][j] - (top == -INFINITY ? 0.f : top));
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) o[t][s][j] *= f, o[t][s][j + 2] *= f;
            }
        const auto place = [&](int t, int s, int j) {  // of o[t][s][j] within a warp's results
            const int r = lane >> 2;
            const int d = 16 * s + (E4M3 ? 2 * r + (j >> 1) : r + 8 * (j >> 1));
            return (8 * t + 2 * (lane & 3) + (j & 1)) * S::PITCH + d;
        };
        if (S::RED < W) {
            if (warp >= S::RED) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) red[(warp - S::RED) * S::HEADS * S::PITCH + place(t, s, j)] = o[t][s][j];
            }
            __syncthreads();
            if (warp < W - S::RED) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[t][s][j] += red[warp * S::HEADS * S::PITCH + place(t, s, j)];
            }
        }
        if (warp < S::RED) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) red[warp * S::HEADS * S::PITCH + place(t, s, j)] = o[t][s][j];
        }
        __syncthreads();
        const auto block_stats = [&](int h) {  // largest logit and sum over the block's warps
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w * S::HEADS + h].x);
            const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < W; ++w) sum += stats[w * S::HEADS + h].y * exp2f(stats[w * S::HEADS + h].x - from);
            return make_float2(top, sum);
        };
        const auto block_sum = [&](int h, int d) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < S::RED; ++w) {
                const float4 x = *reinterpret_cast<const float4 *>(red + (w * S::HEADS + h) * S::PITCH + d);
                v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
            }
            return v;
        };

        const int64_t segment_start = u0 + done - unit, segment_end = segment_start + seen.units;
        const int n4 = heads * a.dim / 4;
        if (piece == seen.units) {  // all of it
            for (int e = threadIdx.x; e < (n4 + 31) / 32 * 32; e += S::THREADS) {
                const bool there = e < n4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (there) {
                    const int h = 4 * e / a.dim;
                    const float2 st = block_stats(h);
                    const float f = inverse_sum(st.y) * a.v_scale;
                    v = block_sum(h, 4 * e - h * a.dim);
                    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
                }
                write_output(a, row, head0, 4 * e, v, there);
            }
            if (WEIGHTS) {
                for (int h = threadIdx.x; h < heads; h += S::THREADS) {
                    const float2 st = block_stats(h);
                    a.norms[(int64_t)row * a.q_heads + head0 + h] = make_float2(st.x, inverse_sum(st.y) * P::UP);
                }
            }
        } else {
            float *part = a.parts + (int64_t)(2 * blockIdx.x + (unit == 0 ? 1 : 0)) * S::PART;
            for (int e = threadIdx.x; e < n4; e += S::THREADS) {
                const int h = 4 * e / a.dim, d = 4 * e - h * a.dim;
                __stcg(reinterpret_cast<float4 *>(part + h * DP + d), block_sum(h, d));
            }
            for (int h = threadIdx.x; h < heads; h += S::THREADS) {
                const float2 st = block_stats(h);
                __stcg(part + S::HEADS * DP + h, st.x);
                __stcg(part + S::HEADS * DP + S::HEADS + h, st.y);
            }
            __threadfence();
            __syncthreads();
            const int first = (int)(segment_start / per_block), last = (int)((segment_end - 1) / per_block);
            if (threadIdx.x == 0) {
                int *counter = a.counters + (int64_t)row * segments_row + segment;
                is_last = atomicAdd(counter, 1) == last - first;
                if (is_last) *counter = 0;  // for the next call
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                const int n_parts = last - first + 1;
                const auto part_of = [&](int i) { return a.parts + (int64_t)(2 * (first + i) + (i == 0 ? 1 : 0)) * S::PART; };
                // factors of the parts, over the warps' results
                float *factor = red;
                for (int i = threadIdx.x; i < n_parts * heads; i += S::THREADS) {
                    const int n = i / heads, h = i - n * heads;
                    factor[n * S::HEADS + h] = __ldcg(part_of(n) + S::HEADS * DP + h);
                }
                __syncthreads();
                for (int h = warp; h < heads; h += W) {
                    float top = -INFINITY, sum = 0.f;
                    for (int n = lane; n < n_parts; n += 32) top = fmaxf(top, factor[n * S::HEADS + h]);
#pragma unroll
                    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
                    const float from = top == -INFINITY ? 0.f : top;
                    for (int n = lane; n < n_parts; n += 32) {
                        const float f = exp2f(factor[n * S::HEADS + h] - from);
                        sum += f * __ldcg(part_of(n) + S::HEADS * DP + S::HEADS + h);
                        factor[n * S::HEADS + h] = f;
                    }
#pragma unroll
                    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
                    const float inv = inverse_sum(sum);
                    for (int n = lane; n < n_parts; n += 32) factor[n * S::HEADS + h] *= inv * a.v_scale;
                    if (WEIGHTS && lane == 0) a.norms[(int64_t)row * a.q_heads + head0 + h] = make_float2(top, inv * P::UP);
                }
                __syncthreads();
                for (int e = threadIdx.x; e < (n4 + 31) / 32 * 32; e += S::THREADS) {
                    const bool there = e < n4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (there) {
                        const int h = 4 * e / a.dim, d = 4 * e - h * a.dim;
#pragma unroll 8
                        for (int n = 0; n < n_parts; ++n) {
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(part_of(n) + h * DP + d));
                            const float f = factor[n * S::HEADS + h];
                            v = make_float4(v.x + f * x.x, v.y + f * x.y, v.z + f * x.z, v.w + f * x.w);
                        }
                    }
                    write_output(a, row, head0, 4 * e, v, there);
                }
            }
        }
        __syncthreads();  // the results' place is free for the next piece

        done += piece;
        unit += piece;
        if (done < count && unit == seen.units) {
            unit = 0;
            if (++segment == segments_row) {
                segment = 0;
                do {
                    seen = row_of(a, ++row);
                } while (seen.units == 0);
            }
        }
    }
}

// Adds to every seen token's weight what its query heads gave it.  A thread a token; the logits of the attention kernel are read once.
__global__ void __launch_bounds__(256) attention_weights_kernel(const AttnArgs a, float *weights, int64_t weights_stride, int64_t weights_len) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.z, kv_head = blockIdx.y;
    const Row r = row_of(a, row);
    const float2 *norms = a.norms + (int64_t)row * a.q_heads + kv_head * a.group;
    const int64_t end = min((int64_t)r.end, weights_len);
    for (int64_t key = r.first + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; key < end; key += (int64_t)gridDim.x * blockDim.x) {
        const float *s = a.logits + (((int64_t)row * a.kv_heads + kv_head) * a.positions + key) * a.group;
        float given = 0.f;
        for (int h = 0; h < a.group; ++h) given += exp2f(s[h] - norms[h].x) * norms[h].y;
        weights[((int64_t)row * a.kv_heads + kv_head) * weights_stride + key] += given;
    }
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

struct Workspace {
    size_t parts, norms, logits, total;
};
int workspace_of(int64_t rows, int64_t q_heads, const jq_kv_cache *c, bool weights, Workspace *w) {
    DeviceCaps caps;
    if (int rc = device_caps(&caps)) return rc;
    w->parts = rounded(JQ_PAGED_ATTENTION_COUNTERS(rows, q_heads));
    const size_t part = 16 * 256 + 32;  // floats, the widest
    w->norms = w->parts + rounded(2 * (size_t)caps.sm_count * part * sizeof(float));
    w->logits = w->norms + (weights ? rounded(sizeof(float2) * (size_t)rows * q_heads) : 0);
    w->total = w->logits + (weights ? rounded(sizeof(float) * (size_t)rows * q_heads * (size_t)(c->max_pages * c->page_size)) : 0);
    return JQ_OK;
}

template <typename T, int DP, int NT, bool WEIGHTS>
int launch_as(cudaStream_t st, AttnArgs &a, int blocks) {
    using S = Shape<T, DP, NT>;
    const auto kernel = paged_attention_kernel<T, DP, NT, WEIGHTS>;
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::SMEM)) return rc;
    a.tiles = (a.group + S::HEADS - 1) / S::HEADS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, (const AttnArgs)a));
    return JQ_OK;
}

template <typename T, bool WEIGHTS>
int launch_for(cudaStream_t st, AttnArgs &a, int blocks) {
    if (a.dim > 128) return launch_as<T, 256, 1, WEIGHTS>(st, a, blocks);
    if (a.group > 8) return a.dim > 64 ? launch_as<T, 128, 2, WEIGHTS>(st, a, blocks) : launch_as<T, 64, 2, WEIGHTS>(st, a, blocks);
    return a.dim > 64 ? launch_as<T, 128, 1, WEIGHTS>(st, a, blocks) : launch_as<T, 64, 1, WEIGHTS>(st, a, blocks);
}

template <bool WEIGHTS>
int launch_type(cudaStream_t st, AttnArgs &a, int type, int blocks) {
    if (type == JQ_KV_F16) return launch_for<KvF16, WEIGHTS>(st, a, blocks);
    if (type == JQ_KV_BF16) return launch_for<KvBf16, WEIGHTS>(st, a, blocks);
    return launch_for<KvE4m3, WEIGHTS>(st, a, blocks);
}

int check_heads(int64_t rows, int64_t q_heads, const jq_kv_cache *c) {
    if (rows < 0 || q_heads <= 0) return set_error(JQ_ERR_INVALID_ARG, "attention: a size is not positive");
    if (q_heads % c->num_kv_heads != 0)
        return set_error(JQ_ERR_SHAPE, "attention: %lld query heads do not divide among %lld key heads", (long long)q_heads, (long long)c->num_kv_heads);
    if (rows > 0x7FFFFFF || q_heads > 65535) return set_error(JQ_ERR_TOO_LARGE, "attention: too many rows or heads");
    return JQ_OK;
}

}  // namespace

}  // namespace jq

using namespace jq;

extern "C" {

size_t jq_paged_attention_ws_bytes(int64_t num_rows, int64_t num_q_heads, const jq_kv_cache *cache, int weights) {
    KvIndex ix;
    Workspace w;
    if (check_kv_cache(cache, &ix) || check_heads(num_rows, num_q_heads, cache) || workspace_of(num_rows, num_q_heads, cache, weights != 0, &w))
        return 0;
    return w.total;
}

int jq_paged_attention_q8_1_device(void *stream, const float *d_q, int64_t q_stride_row, int64_t q_stride_head, int64_t num_rows,
                                   int64_t num_q_heads, const jq_kv_cache *cache, const int32_t *d_lens, const int32_t *d_seqs,
                                   float scale, int64_t window, float *d_out, void *d_xq, int order, int s_mode, float *d_weights,
                                   int64_t weights_stride, int64_t weights_len, void *d_ws, size_t ws_bytes) {
    AttnArgs a = {};
    if (int rc = check_kv_cache(cache, &a.ix)) return rc;
    if (int rc = check_heads(num_rows, num_q_heads, cache)) return rc;
    if (window < 0) return set_error(JQ_ERR_INVALID_ARG, "attention: negative window");
    if (!std::isfinite(scale)) return set_error(JQ_ERR_INVALID_ARG, "attention: scale is not finite");
    if (d_out == nullptr && d_xq == nullptr) return set_error(JQ_ERR_INVALID_ARG, "attention: no output requested");
    const int64_t dim = cache->head_dim;
    if (d_xq != nullptr) {
        if (order != JQ_ORDER_KSUPER_COL && order != JQ_ORDER_COL_KSUPER) return set_error(JQ_ERR_INVALID_ARG, "unknown Q8_1 block order %d", order);
        if (s_mode != JQ_S_SUM_X && s_mode != JQ_S_D_SUM_Q) return set_error(JQ_ERR_INVALID_ARG, "unknown s_mode %d", s_mode);
        if (dim % QK != 0 || num_q_heads * dim % SUPER != 0)
            return set_error(JQ_ERR_UNSUPPORTED, "attention with Q8_1 output needs head_dim %% 32 == 0 and num_q_heads * head_dim %% 128 == 0");
    }
    if (d_seqs == nullptr && num_rows > cache->num_seqs)
        return set_error(JQ_ERR_INVALID_ARG, "attention: %lld rows, and %lld sequences", (long long)num_rows, (long long)cache->num_seqs);
    if (d_weights != nullptr) {
        if (d_seqs != nullptr) return set_error(JQ_ERR_UNSUPPORTED, "attention: weights are kept per sequence: one row each, d_seqs NULL");
        if (num_rows > 65535) return set_error(JQ_ERR_TOO_LARGE, "attention: more than 65535 rows with weights");
        if (weights_len < 0 || weights_stride < weights_len) return set_error(JQ_ERR_INVALID_ARG, "attention: rows of the weights overlap");
    }
    if (num_rows == 0) return JQ_OK;
    if (d_q == nullptr || d_lens == nullptr || d_ws == nullptr) return set_error(JQ_ERR_INVALID_ARG, "attention: null pointer");
    const uintptr_t bits = (uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_xq | (uintptr_t)d_ws | (uintptr_t)(4 * q_stride_row) | (uintptr_t)(4 * q_stride_head);
    if ((bits & 15u) != 0) return set_error(JQ_ERR_ALIGN, "attention: queries, outputs and workspace must be 16-byte aligned");
    if ((((uintptr_t)d_lens | (uintptr_t)d_seqs | (uintptr_t)d_weights) & 3u) != 0)
        return set_error(JQ_ERR_ALIGN, "attention: lengths, sequences and weights must be 4-byte aligned");
    Workspace w;
    if (int rc = workspace_of(num_rows, num_q_heads, cache, d_weights != nullptr, &w)) return rc;
    if (ws_bytes < w.total)
        return set_error(JQ_ERR_INVALID_ARG, "attention: a workspace of %zu bytes is needed, %zu given", w.total, ws_bytes);
    DeviceCaps caps;
    if (int rc = device_caps(&caps)) return rc;
    const int blocks = caps.sm_count < MAX_BLOCKS ? caps.sm_count : MAX_BLOCKS;
    a.q = d_q, a.q_row = q_stride_row, a.q_head = q_stride_head;
    a.k = static_cast<const char *>(cache->d_k), a.v = static_cast<const char *>(cache->d_v);
    a.lens = d_lens, a.seqs = d_seqs, a.out = d_out, a.xq = static_cast<uint8_t *>(d_xq);
    a.scale_log2 = (float)((double)scale * cache->k_scale * 1.4426950408889634);
    a.v_scale = cache->v_scale;
    a.rows = (int)num_rows, a.q_heads = (int)num_q_heads, a.kv_heads = (int)cache->num_kv_heads, a.group = a.q_heads / a.kv_heads, a.dim = (int)dim;
    a.positions = cache->max_pages * cache->page_size;
    a.window = window >= a.positions ? 0 : (int)window;
    a.n_super = (int)(num_q_heads * dim / SUPER), a.order = order, a.s_mode = s_mode;
    char *ws = static_cast<char *>(d_ws);
    a.counters = reinterpret_cast<int *>(ws);
    a.parts = reinterpret_cast<float *>(ws + w.parts);
    a.norms = reinterpret_cast<float2 *>(ws + w.norms);
    a.logits = reinterpret_cast<float *>(ws + w.logits);
    a.fault = device_fault_ptr();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d_weights == nullptr) return launch_type<false>(st, a, cache->type, blocks);
    if (int rc = launch_type<true>(st, a, cache->type, blocks)) return rc;
    if (a.positions == 0) return JQ_OK;
    int64_t across = (a.positions + 255) / 256;
    if (across > 64) across = 64;  // a block walks on where sequences are longer
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)across, (unsigned)a.kv_heads, (unsigned)num_rows);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attention_weights_kernel, (const AttnArgs)a, d_weights, weights_stride, weights_len));
    return JQ_OK;
}

}  // extern "C"
