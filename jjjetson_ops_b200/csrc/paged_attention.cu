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
// with a 16-bit element are exact, and the sums are fp32.  fp16 has few exponents: of a query's elements what is rounded away is up to 2^-24 of
// their largest, of a probability up to 2^-23 of itself or 2^-40 of the row's largest, whichever is more.  So the n keys of a long row that have
// next to nothing are together off by n 2^-40 of the largest value at most (a million: 2^-20); the sum of probabilities has them whole.
//
// The work is cut into units of 16 keys of one row and key head, all units of the call laid end to end, and every warp takes an equal
// stretch: long and short rows need no plan on the host, and lengths stay on the device.  A warp needs no other one until its stretch
// is done: it has a ring of tiles of its own (asynchronous 16-byte copies), which runs on across the ends of rows, and what it has of a
// row that begins or ends with another warp it leaves in shared memory.  Then the block puts those parts together, and where a row goes
// on in another block leaves its part in the workspace; the block that finds itself the last of a row's adds the parts, in their order,
// so the result does not depend on who came last.
#include "kv_cache.cuh"

#include <cmath>

namespace jq {

namespace {

constexpr int UNIT = 16;          // keys; what the work is divided by
// What a warp spends on the beginning of a segment (its queries, and what it had of the one before into shared memory), in units: stretches are
// equal with this counted in.  Without it the warps of a block that had one segment more were done 6 us later (16 sequences of up to
// 2500 tokens, 32 key heads).
constexpr int BEGIN = 5;
constexpr int STEP = 2;           // units that a warp takes at a time: two tiles of 16 rows for the tensor cores
constexpr int SMEM_BYTES = 227 * 1024;

struct AttnArgs {
    const float *q;
    int64_t q_row, q_head;
    const char *k, *v;
    KvIndex ix;
    const int32_t *lens, *seqs;
    float *out;
    uint8_t *xq;
    float scale;       // times 2^scale_exponent: scale * k_scale / ln 2.  Zero, or its size is in [1, 2]
    int scale_exponent;
    float v_scale;
    int rows, q_heads, kv_heads, group, dim, window;
    int tiles;         // parts of a group that are computed apart (groups of more heads than one pass takes)
    int n_super, order, s_mode;
    // workspace
    int *counters;     // one for every segment that blocks share: never more than there are blocks
    float *parts;
    float2 *norms;     // [rows][q_heads]: largest logit, 1 / sum (with weights)
    float *logits;     // [rows][kv_heads][positions][group] (with weights)
    int positions;     // that a row of the page table has room for
    bool grouped;      // pages hold whole units
    int *fault;
};

// ---- element types: how 16 keys x 16 elements become operands ---------------------------------------------
// d += a b, or d = a b
#define JQ_MMA(name, types)                                                                                                              \
    __device__ __forceinline__ void name(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {                                \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." types ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                  \
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                                             \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));                                                         \
    }                                                                                                                                    \
    __device__ __forceinline__ void name##_first(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {                        \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." types ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"              \
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                                             \
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));                                               \
    }
JQ_MMA(mma_f16, "f16.f16")
JQ_MMA(mma_bf16, "bf16.bf16")
#undef JQ_MMA
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
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
    static constexpr float UP = 32768.f;  // probabilities, which are 1 at most, are held times 2^15: the most that fp16 has room for
    static constexpr int ROOM = 0, MOST = 100;  // see the queries: a product is below 4 * 2^16 * 256 = 2^26
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&w)[N]) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
        w[0] = *reinterpret_cast<const uint32_t *>(&h);
        w[1] = *reinterpret_cast<const uint32_t *>(&l);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], bool first) { first ? mma_f16_first(d, a, b) : mma_f16(d, a, b); }
};
template <>
struct Parts<KvE4m3> : Parts<KvF16> {};  // e4m3 elements become fp16, exactly
template <>
struct Parts<KvBf16> {
    static constexpr int N = 3;
    static constexpr float UP = 1.f;
    static constexpr int ROOM = 16, MOST = 127;  // with keys up to 2^128 a product is below 2^-14 * 2^128 * 256 = 2^122
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&w)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            const float2 f = __bfloat1622float2(h);
            a -= f.x, b -= f.y;
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], bool first) { first ? mma_bf16_first(d, a, b) : mma_bf16(d, a, b); }
};

// the two pairs of e4m3 in a register as two pairs of fp16
__device__ __forceinline__ void halves_of_e4m3(uint32_t four, uint32_t &low, uint32_t &high) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(low), "=r"(high) : "r"(four));
}
// 2^x to 2^-22 of its value; 0 for -infinity and for what is below 2^-126
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One warp's part of a piece, by its place in the order: where the piece lies, and where the part does.
struct Entry {
    int row, segment, unit, n, units;  // units [unit, unit + n) of the row's
    int start;                         // where the segment begins, from the block's beginning on
};

// Shapes of one instance.
template <typename T, int DP_, int NT_>
struct Shape {
    static constexpr int DP = DP_;                  // head_dim, padded
    static constexpr int NT = NT_;                  // tiles of eight heads
    static constexpr int HEADS = 8 * NT;
    // A warp's accumulators and queries fill its registers.  8-bit tiles are half as long on their way and need conversion: twelve warps (168
    // registers) where they fit, eight of them 110 us against 98 for 64 sequences of up to 5000 tokens.  Sixteen heads in one pass, or 8-bit
    // heads of 256: eight warps with two tiles each and not four with six (20 sequences of up to 3000 tokens, 64 heads on 4, 31.8 us against
    // 38.6; two of 93548 on e4m3, 16 heads on one, 44.6 against 69.6).  16-bit heads of 256 leave room for four.
    static constexpr int WARPS = DP == 256 && sizeof(typename T::Element) == 2 ? 4 : sizeof(typename T::Element) == 1 && NT == 1 && DP == 128 ? 12 : 8;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ROW = DP * (int)sizeof(typename T::Element);  // bytes
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int KEYS = STEP * UNIT;
    static constexpr int TILE = KEYS * ROW;         // keys, or values, of a step
    static constexpr int RESULT = HEADS * DP * 4 + HEADS * 8;  // a warp's result: sums, then per head the largest logit and the sum of weights
    static constexpr int FIXED = WARPS * (RESULT + 2 * (int)sizeof(Entry) + 32) + 32;
    static constexpr int FIT = (SMEM_BYTES - FIXED) / (WARPS * TILE);
    static constexpr int SLOTS = FIT < 6 ? FIT : 6;
    static constexpr int RING = WARPS * SLOTS * TILE;
    static constexpr int SMEM = RING + FIXED;
    static constexpr int PART = HEADS * DP + 2 * HEADS;  // floats of a part: as a result
    static constexpr int CHAINS = NT == 1 ? Parts<T>::N : 2;  // sums of a logit: one per part of the queries, so that they are made side by side
    static constexpr bool EARLY_QUERIES = NT * DP <= 128 && WARPS <= 8;  // the others' registers are full
    static constexpr int LEAST = WARPS * STEP;      // units of a block at least: a step for every warp
    static_assert(SLOTS >= 2, "while one tile is read another is on its way");
    static_assert(SLOTS * TILE >= RESULT + 2 * WARPS * HEADS * 12, "a warp's last result takes the place of its ring, the block's factors what is behind it");
    static_assert(2 * WARPS * HEADS <= THREADS, "a thread for every factor");
};

// Where element `d` of head `h` of a result lies: eight rows' eight elements in different banks, four elements together.
template <int DP>
__device__ __forceinline__ int result_at(int h, int d) {
    return h * DP + (d ^ ((h >> 1 & 3) << 3));
}

// Within a tile the 16-byte chunks of a row are spread so that eight rows' same chunk lies in different banks: chunk c of row r lies at
// c ^ spread(r).  Addresses of other chunks and rows follow from a lane's own by constants: an exclusive or within the row (tiles begin at
// multiples of a row), then an addition.
template <int CHUNKS>
__device__ __forceinline__ constexpr int spread(int r) {
    return CHUNKS >= 8 ? (r & 7) : ((r >> 1) & (CHUNKS - 1));
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
    r.end = r.seq < 0 ? 0 : max(0, min(a.lens[row], a.positions));
    r.first = a.window > 0 && r.end > a.window ? r.end - a.window : 0;
    r.unit0 = r.first / UNIT;
    r.units = r.end > 0 ? (r.end + UNIT - 1) / UNIT - r.unit0 : 0;
    return r;
}

// Inclusive sum over the warp.
__device__ __forceinline__ uint32_t warp_inclusive(uint32_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
// Rows lie end to end, `count(row)` things each: the row in which thing `at` lies, and how many are before it there.  Every warp looks for
// itself (no barrier); `own`: the row of the lane's number, `at` is below the sum (else the row is nonsense, and within the table).
template <typename F>
__device__ __forceinline__ int find_row(const AttnArgs &a, const Row &own, uint32_t at, F &&count, uint32_t *within) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int r0 = 0;; r0 += 32) {
        const uint32_t n = r0 + lane < a.rows ? (uint32_t)count(r0 == 0 ? own : row_of(a, r0 + lane)) : 0;
        const uint32_t end = warp_inclusive(n);
        const uint32_t behind = __ballot_sync(0xFFFFFFFFu, at < end);
        if (behind != 0 || r0 + 32 >= a.rows) {
            const int i = behind != 0 ? __ffs(behind) - 1 : 0;
            *within = at - __shfl_sync(0xFFFFFFFFu, end - n, i);
            return r0 + i;
        }
        at -= __shfl_sync(0xFFFFFFFFu, end, 31);
    }
}
__device__ __forceinline__ Row row_at(const AttnArgs &a, const Row &own, int row) {
    if (row >= 32) return row_of(a, row);
    Row r;
    r.seq = __shfl_sync(0xFFFFFFFFu, own.seq, row);
    r.first = __shfl_sync(0xFFFFFFFFu, own.first, row);
    r.end = __shfl_sync(0xFFFFFFFFu, own.end, row);
    r.units = __shfl_sync(0xFFFFFFFFu, own.units, row);
    r.unit0 = __shfl_sync(0xFFFFFFFFu, own.unit0, row);
    return r;
}

// Four consecutive elements of the output: element `e` of the heads of one key head's tile (their elements lie end to end), as
// fp32 and as Q8_1.  Every lane of the warp calls it, with consecutive e; `there`: it has elements.  (The quantizer is some 200 instructions,
// and called from several places.)
__device__ __noinline__ void write_q8(uint8_t *xq, int n, int row, int n_super, int rows, int order, int s_mode, float4 v, bool there) {
    if (!there) v = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t ds;
    const uint32_t q = quantize_group_q8_1(v, s_mode, &ds);
    if (there) {
        uint8_t *block = xq + q8_block_index(n / SUPER, row, n_super, rows, order) * Q8_BYTES;
        const int i = n % SUPER;
        *reinterpret_cast<uint32_t *>(block + Q8_QS_OFFSET + i) = q;
        if (i % QK == 0) *reinterpret_cast<uint32_t *>(block + i / QK * 4) = ds;
    }
}
__device__ __forceinline__ void write_output(const AttnArgs &a, int row, int head0, int e, float4 v, bool there) {
    const int n = head0 * a.dim + e;  // within the row
    if (a.out != nullptr && there) *reinterpret_cast<float4 *>(a.out + (int64_t)row * a.q_heads * a.dim + n) = v;
    if (a.xq != nullptr) write_q8(a.xq, n, row, a.n_super, a.rows, a.order, a.s_mode, v, there);
}

// What the weights go by: a row whose pages are all bad has logits of minus infinity, which 0 and not their maximum is taken from (times 0, a
// difference of infinities would leave NaN in the weights).
__device__ __forceinline__ float2 norm_of(float top, float inverse) { return make_float2(top == -INFINITY ? 0.f : top, inverse); }
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }  // a row whose pages are all bad gives zeros

template <typename T, int DP, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(Shape<T, DP, NT>::THREADS, 1) paged_attention_kernel(const AttnArgs a) {
    using S = Shape<T, DP, NT>;
    using P = Parts<T>;
    using E = typename T::Element;
    constexpr bool E4M3 = sizeof(E) == 1;
    constexpr int W = S::WARPS;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *results = smem + S::RING;  // one per warp: of a row that began with another warp
    Entry *entries = reinterpret_cast<Entry *>(results + W * S::RESULT);  // two per warp: that, and its last piece
    uint32_t *masks = reinterpret_cast<uint32_t *>(entries + 2 * W);
    int *is_last = reinterpret_cast<int *>(masks + 8 * W);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int segments_row = a.kv_heads * a.tiles;  // a row's key heads, or tiles of their query heads: each has the row's units

    // ---- the block's stretch ----
    Row own = {-1, 0, 0, 0, 0};  // the row of this lane's number
    if (lane < a.rows) own = row_of(a, lane);
    const auto weight_of = [&](const Row &r) { return r.units > 0 ? r.units + BEGIN : 0; };  // of one of its segments
    uint32_t total = own.units * segments_row, segments = own.units > 0 ? segments_row : 0;
#pragma unroll 1
    for (int r = lane + 32; r < a.rows; r += 32) {
        const uint32_t n = row_of(a, r).units;
        total += n * segments_row;
        segments += n > 0 ? segments_row : 0;
    }
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    segments = __reduce_add_sync(0xFFFFFFFFu, segments);
    // Few segments: each gets blocks of its own, so that a block has one segment to put together; at most an eighth of the blocks stay
    // idle.  Many: equal stretches.
    const bool apart = segments <= gridDim.x / 8;
    if (!apart) total += segments * BEGIN;
    uint32_t per_block = apart ? (total + gridDim.x - segments - 1) / (gridDim.x - segments) : (total + gridDim.x - 1) / gridDim.x;
    if (per_block < S::LEAST) per_block = S::LEAST;
    const uint32_t u0 = blockIdx.x * per_block;  // (not apart)
    int count = 0;                               // units of this block
    int first_block = 0, parts_apart = 1;
    struct {
        Row row;
        int r, segment, unit;
    } piece = {};  // the warp's first
    int a0 = 0, a1 = 0;  // the warp's stretch within the block's
    // Apart, the warps take the steps of the block's stretch in turn: eight streams a block through memory instead of one took
    // 98 us for a sequence of 131071 tokens where this takes 93.
    const int hop = apart ? W * STEP : STEP;
    if (apart) {
        uint32_t within;
        piece.r = find_row(a, own, blockIdx.x, [&](const Row &r) { return segments_row * ((r.units + per_block - 1) / per_block); }, &within);
        if (piece.r < a.rows) {
            piece.row = row_at(a, own, piece.r);
            parts_apart = (piece.row.units + per_block - 1) / per_block;
            if (within < (uint32_t)(segments_row * parts_apart)) {
                piece.segment = within / parts_apart;
                const int part = within - piece.segment * parts_apart;
                const int each = (piece.row.units + parts_apart - 1) / parts_apart;
                first_block = blockIdx.x - part;
                piece.unit = part * each;
                count = max(0, min(piece.row.units - piece.unit, each));
                parts_apart = (piece.row.units + each - 1) / each;  // (rounded up, `each` may leave nothing to the last blocks)
            }
        }
        piece.unit += warp * STEP;
        a1 = max(0, count - warp * STEP);
    }

    // ---- the warp's pieces: first those that begin and end with it, then the one that began before, then the last ----
    // (so that what it has of the first piece stays where the others' results were turned around)
    Entry *mine = entries + 2 * warp;  // [0]: the first piece where others follow, [1]: the last; n = 0: none
    Entry first_piece = {piece.r, piece.segment, piece.unit, a1, piece.row.units, 0}, last_piece = first_piece;
    first_piece.n = 0;
    if (!apart && u0 < total) {
        count = min(per_block, total - u0);
        a0 = warp * count / W, a1 = (warp + 1) * count / W;
        if (a0 < a1) {
            const auto find = [&](int at, Entry &e) {  // the segment at `at`, and which of its units begins there
                uint32_t within;
                e.row = find_row(a, own, u0 + at, [&](const Row &r) { return segments_row * weight_of(r); }, &within);
                e.units = __shfl_sync(0xFFFFFFFFu, own.units, e.row & 31);
                if (e.row >= 32) e.units = row_of(a, e.row).units;
                e.segment = within / (e.units + BEGIN);
                e.unit = within - e.segment * (e.units + BEGIN);
                e.start = at - e.unit;
                e.unit = max(0, e.unit - BEGIN);
            };
            find(a0, first_piece);
            find(a1, last_piece);  // (at the call's end: nonsense, and not looked at)
            const bool to_the_end = u0 + a1 >= total;
            if (!to_the_end && last_piece.row == first_piece.row && last_piece.segment == first_piece.segment) {
                first_piece.n = last_piece.unit - first_piece.unit;
                last_piece = first_piece;
                first_piece.n = 0;
            } else {
                first_piece.n = first_piece.units - first_piece.unit;
                last_piece.n = to_the_end ? 0 : last_piece.unit;
                if (to_the_end) last_piece.row = a.rows;
                last_piece.unit = 0;
            }
        } else {
            last_piece.n = 0;
        }
    }
    if (lane == 0) mine[0] = first_piece, mine[1] = last_piece;
    __syncwarp();
    const bool any = first_piece.n > 0 || last_piece.n > 0;
    // A walk over the pieces; `row` and the others of the piece are what the walker needs of it.
    enum { MIDDLE, FIRST, LAST, DONE };
    struct Walk {
        Row row;
        int r, segment, unit, n;  // units left of the piece, from `unit` on
        int phase;
    };
    const auto next_piece = [&](Walk &w) {
        if (w.phase == MIDDLE) {  // the next segment, all of it, if it is not the one that the last piece is of
            if (++w.segment == segments_row) {
                w.segment = 0;
#pragma unroll 1
                do {
                    ++w.r;
                    if (w.r < a.rows) w.row = row_of(a, w.r);
                } while (w.r < a.rows && w.row.units == 0);
            }
            w.unit = 0;
            w.n = w.row.units;
            if (w.r < a.rows && (w.r != mine[1].row || w.segment != mine[1].segment)) return;
        }
        ++w.phase;
        if (w.phase == LAST && mine[1].n == 0) w.phase = DONE;
        if (w.phase != DONE) {
            const Entry &e = mine[w.phase == FIRST ? 0 : 1];
            w.r = e.row, w.segment = e.segment, w.unit = e.unit, w.n = e.n;
            w.row = row_of(a, w.r);
        }
    };
    Walk at, next;  // what is computed, and what is copied
    at.row = row_at(a, own, any ? first_piece.row : 0), at.r = first_piece.row, at.segment = first_piece.segment;
    at.phase = !any ? LAST : first_piece.n > 0 ? MIDDLE : FIRST;  // (the phase before that of the first piece to take)
    next_piece(at);
    next = at;

    // queries of one piece: the elements that go with the keys' operands, 2i, 2i + 1, 2i + 8, 2i + 9 of 16, or with e4m3 the four from
    // 4i on.  They are asked for early where there are registers: before the cache is looked up, and before the piece ahead is put away.
    float raw[NT][DP / 16][4];
    const auto ask_queries = [&]() {
        const int kv_head = a.tiles == 1 ? at.segment : at.segment / a.tiles, tile = at.segment - kv_head * a.tiles;
        const int head0 = kv_head * a.group + tile * S::HEADS, heads = min(S::HEADS, a.group - tile * S::HEADS);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int h = 8 * t + (lane >> 2), i = lane & 3;
            const float *from = a.q + (int64_t)at.r * a.q_row + (int64_t)(head0 + h) * a.q_head;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const bool there = h < heads && 16 * s < a.dim;
                if (E4M3) {
                    const float4 v = there ? *reinterpret_cast<const float4 *>(from + 16 * s + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
                    raw[t][s][0] = v.x, raw[t][s][1] = v.y, raw[t][s][2] = v.z, raw[t][s][3] = v.w;
                } else {
                    const float2 v = there ? *reinterpret_cast<const float2 *>(from + 16 * s + 2 * i) : make_float2(0.f, 0.f);
                    const float2 u = there ? *reinterpret_cast<const float2 *>(from + 16 * s + 2 * i + 8) : make_float2(0.f, 0.f);
                    raw[t][s][0] = v.x, raw[t][s][1] = v.y, raw[t][s][2] = u.x, raw[t][s][3] = u.y;
                }
            }
        }
    };
    if (S::EARLY_QUERIES && any) ask_queries();

    // ---- the ring: tiles of keys and of values in turn ----
    // A step's keys lie in pages.  Where a page holds whole units, every lane has the two units' offsets, else each lane has its own
    // key's, and they are passed around.
    unsigned char *const my_ring = smem + warp * S::SLOTS * S::TILE;
    const uint32_t ring = smem_u32(my_ring);
    uint32_t *mask_ring = masks + warp * S::SLOTS;
    const bool grouped = a.grouped;
    // What the page table was asked for the step that is copied next; the answer is looked at half a step later.
    struct {
        int key0;
        uint32_t mask;     // which of the 32 keys are there
        int page[2];
        int64_t head;
        bool live;         // a step, even if none of its keys is
    } asked;
    const auto ask = [&]() {
        asked.live = next.phase != DONE;
        if (!asked.live) return;
        const int key0 = (next.row.unit0 + next.unit) * UNIT;
        const int end = min(next.row.end, key0 + min(next.n, STEP) * UNIT);
        const int32_t *table = a.ix.table + (int64_t)next.row.seq * a.ix.table_stride;
        const uint32_t from = next.row.first > key0 ? 0xFFFFFFFFu << (next.row.first - key0) : 0xFFFFFFFFu;
        const uint32_t until = end - key0 >= 32 ? 0xFFFFFFFFu : ~(0xFFFFFFFFu << (end - key0));
        asked.key0 = key0;
        asked.mask = from & until;
        asked.head = (int64_t)(a.tiles == 1 ? next.segment : next.segment / a.tiles) * a.ix.stride_head;
        asked.page[0] = asked.page[1] = 0;
        if (grouped) {
            asked.page[0] = table[kv_page_of(a.ix, (uint32_t)key0)];
            if (key0 + UNIT < end) asked.page[1] = table[kv_page_of(a.ix, (uint32_t)(key0 + UNIT))];
        } else if (asked.mask >> lane & 1u) {
            asked.page[0] = table[kv_page_of(a.ix, (uint32_t)(key0 + lane))];
        }
        next.unit += hop;
        next.n -= hop;
        if (next.n <= 0) next_piece(next);
    };
    const int my_chunk = lane % S::CHUNKS;
    const bool inside = my_chunk * 16 < a.dim * (int)sizeof(E);
    constexpr int AT_ONCE = 32 / S::CHUNKS;  // rows that the warp copies with one instruction
    const uint32_t my_place = lane / S::CHUNKS * S::ROW + (my_chunk ^ spread<S::CHUNKS>(lane / S::CHUNKS)) * 16;
    // of the operands that this lane reads: keys (rows of the product are keys) and values (rows are elements)
    const uint32_t k_place = (lane & 15) * S::ROW + ((lane >> 4) ^ spread<S::CHUNKS>(lane & 15)) * 16;
    const uint32_t v_place = ((lane & 7) + (lane >> 4) * 8) * S::ROW + ((lane >> 3 & 1) ^ spread<S::CHUNKS>(lane & 7)) * 16;
    const int64_t row_stride = a.ix.stride_slot * (int)sizeof(E);
    const int64_t my_start = inside ? (lane / S::CHUNKS) * row_stride + my_chunk * 16 : 0;
    struct {
        int64_t offset[2];  // bytes, of this lane's first rows of the two units (not grouped: of its key)
        uint32_t mask;
        bool live;
    } here = {};
    // Tile 2n is the keys, 2n + 1 the values of the warp's n-th step; tile t lies in slot t % SLOTS.
    int slot_next = S::SLOTS - 1, mask_next = 0;
    const auto copy_next = [&](bool values) {
        if (!values) {
            here.live = asked.live;
            here.mask = asked.mask;
            const uint32_t units = grouped ? 0x0000FFFFu : 1u << lane;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const uint32_t mine_of = g == 0 ? units : ~units;
                const int64_t to = kv_offset(a.ix, (uint32_t)(asked.key0 + (grouped ? UNIT * g : lane)), asked.page[g]);
                here.offset[g] = (to + asked.head) * (int)sizeof(E) + (grouped ? my_start : my_chunk * 16);
                if (to < 0) {
                    here.offset[g] = 0;
                    if (asked.live && (asked.mask & mine_of) != 0 && (grouped || g == 0)) report_bad_page(a.fault);
                    if (grouped) here.mask &= ~mine_of;
                }
                if (!grouped && g == 0) here.mask = __ballot_sync(0xFFFFFFFFu, to >= 0) & asked.mask;
            }
            if (lane == 0) mask_ring[mask_next] = here.mask;
            if (++mask_next == S::SLOTS) mask_next = 0;
        }
        const char *pool = values ? a.v : a.k;
        const uint32_t to = ring + slot_next * S::TILE;
        if (here.live) {
            const uint32_t own = to + my_place;
            if (grouped) {
                const char *from[2] = {pool + here.offset[0], pool + here.offset[1]};
                if (here.mask == 0xFFFFFFFFu) {
#pragma unroll
                    for (int i = 0; i < S::KEYS / AT_ONCE; ++i) {
                        copy16((own ^ (spread<S::CHUNKS>(i * AT_ONCE) * 16)) + i * AT_ONCE * S::ROW, from[i * AT_ONCE / UNIT], inside);
                        from[i * AT_ONCE / UNIT] += AT_ONCE * row_stride;
                    }
                } else {
                    // (a unit that is not there has a place in the pool all the same; it is not read)
                    const uint32_t mine_of = inside ? here.mask >> (lane / S::CHUNKS) : 0;
#pragma unroll
                    for (int i = 0; i < S::KEYS / AT_ONCE; ++i) {
                        const bool there = mine_of >> (i * AT_ONCE) & 1u;
                        copy16((own ^ (spread<S::CHUNKS>(i * AT_ONCE) * 16)) + i * AT_ONCE * S::ROW, there ? from[i * AT_ONCE / UNIT] : pool, there);
                        from[i * AT_ONCE / UNIT] += AT_ONCE * row_stride;
                    }
                }
            } else {
#pragma unroll 4
                for (int i = 0; i < S::KEYS / AT_ONCE; ++i) {
                    const int r = lane / S::CHUNKS + i * AT_ONCE;
                    const int64_t offset = __shfl_sync(0xFFFFFFFFu, here.offset[0], r) - (r % S::CHUNKS) * 16 + my_chunk * 16;  // (with that lane's chunk)
                    const bool there = inside && (here.mask >> r & 1u);
                    copy16((own ^ (spread<S::CHUNKS>(i * AT_ONCE) * 16)) + i * AT_ONCE * S::ROW, pool + (there ? offset : 0), there);
                }
            }
        }
        if (values) ask();
        if (++slot_next == S::SLOTS) slot_next = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // A new tile goes into the slot of the one that was read before, then the oldest is waited for and read.
    constexpr bool SAME = (S::SLOTS & 1) != 0;  // what is copied while keys are read: keys, else values
    asked.live = false;
#pragma unroll 1
    for (int t = -1; t < S::SLOTS - 1; ++t) copy_next(t & 1);  // (the values of a step before the first, which is none: the page table is asked there)
    int slot = 0, mask_slot = 0;
    const auto next_tile = [&](bool values) {
        __syncwarp();
        copy_next(values == SAME);
        asm volatile("cp.async.wait_group %0;" ::"n"(S::SLOTS - 1) : "memory");
        __syncwarp();
        const uint32_t tile = ring + slot * S::TILE;
        if (++slot == S::SLOTS) slot = 0;
        return tile;
    };

#pragma unroll 1
    while (at.phase != DONE) {
        const int kv_head = a.tiles == 1 ? at.segment : at.segment / a.tiles, tile_of = at.segment - kv_head * a.tiles;
        const int head0 = kv_head * a.group + tile_of * S::HEADS, heads = min(S::HEADS, a.group - tile_of * S::HEADS);
        uint32_t q[NT][DP / 16][P::N][2];
        float unscale[NT][2];
        float o[NT][DP / 16][4];
        float m[NT][2], l[NT][2];
        // Queries: two or three operands per 16 elements, times the scale and a power of two so that fp16, or a product with bf16's largest keys,
        // holds them.  What is left of the scale, `unscale`, is a power of two: logits are exact multiples of the products, so that however large
        // they are the largest one's difference from itself is nothing (a rounded factor would leave it off by half a bit of the logit).
        if (!S::EARLY_QUERIES) ask_queries();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float largest = 0.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) largest = fmaxf(largest, fabsf(raw[t][s][j]));
            largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 2));
            // 2^-e with 2^e <= largest (times 2^ROOM), within 2^-126 .. 2^126
            int e = (int)(__float_as_uint(largest) >> 23) - 127 + P::ROOM;
            e = largest == 0.f ? 0 : max(-126, min(126, e));
            const float down = __uint_as_float((uint32_t)(127 - e) << 23) * a.scale;
            // not 0, which a key that is not seen has to be minus infinity times; and no finite product becomes an infinite logit, but with bf16
            e = max(-149, min(P::MOST, e + a.scale_exponent));
            const float up = __uint_as_float(e >= -126 ? (uint32_t)(127 + e) << 23 : 1u << (149 + e));
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                uint32_t w0[P::N], w1[P::N];
                P::split(raw[t][s][0] * down, raw[t][s][1] * down, w0);
                P::split(raw[t][s][2] * down, raw[t][s][3] * down, w1);
#pragma unroll
                for (int j = 0; j < P::N; ++j) q[t][s][j][0] = w0[j], q[t][s][j][1] = w1[j];
            }
            // the products' columns: this lane has heads 2i and 2i + 1
            unscale[t][0] = __shfl_sync(0xFFFFFFFFu, up, 8 * (lane & 3));
            unscale[t][1] = __shfl_sync(0xFFFFFFFFu, up, 8 * (lane & 3) + 4);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t][s][j] = 0.f;
        }

#pragma unroll 1
        for (int u = 0; u < at.n; u += hop) {
            uint32_t tile = next_tile(false);
            const uint32_t mask = mask_ring[mask_slot];
            if (++mask_slot == S::SLOTS) mask_slot = 0;
            uint32_t p[NT][2][P::N][2];
            float shrink[NT][2];
            // logits of 2 x 16 keys x 8 NT heads
            float s4[NT][2][S::CHAINS][4];
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                if constexpr (E4M3) {
                    if (s & 1) continue;
                    uint32_t r[2][4];
#pragma unroll
                    for (int g = 0; g < 2; ++g) ldmatrix4(r[g], ((tile + k_place) ^ (s * 16)) + UNIT * g * S::ROW);
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        uint32_t k8[2][4];
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            halves_of_e4m3(r[g][2 * v], k8[g][0], k8[g][2]);
                            halves_of_e4m3(r[g][2 * v + 1], k8[g][1], k8[g][3]);
                        }
#pragma unroll
                        for (int j = 0; j < P::N; ++j)
#pragma unroll
                            for (int g = 0; g < 2; ++g)
#pragma unroll
                                for (int t = 0; t < NT; ++t) P::mma(s4[t][g][j % S::CHAINS], k8[g], q[t][s + v][j], s + v == 0 && j < S::CHAINS);
                    }
                } else {
                    uint32_t k[2][4];
#pragma unroll
                    for (int g = 0; g < 2; ++g) ldmatrix4(k[g], ((tile + k_place) ^ (s * 32)) + UNIT * g * S::ROW);
#pragma unroll
                    for (int j = 0; j < P::N; ++j)
#pragma unroll
                        for (int g = 0; g < 2; ++g)
#pragma unroll
                            for (int t = 0; t < NT; ++t) P::mma(s4[t][g][j % S::CHAINS], k[g], q[t][s][j], s == 0 && j < S::CHAINS);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                // x: products of the scaled queries; logits in base 2 are x times unscale (a power of two)
                float x[2][4];
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[g][j] = s4[t][g][S::CHAINS - 1][j];
#pragma unroll
                        for (int i = S::CHAINS - 2; i >= 0; --i) x[g][j] += s4[t][g][i][j];
                    }
                if (mask != 0xFFFFFFFFu) {
                    const uint32_t seen = mask >> (lane >> 2);
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[g][j] = seen >> (16 * g + 8 * (j >> 1)) & 1u ? x[g][j] : -INFINITY;
                }
                if (WEIGHTS) {
                    const int kv_head = a.tiles == 1 ? at.segment : at.segment / a.tiles;
                    const int h = (at.segment - kv_head * a.tiles) * S::HEADS + 8 * t + 2 * (lane & 3);
                    const int key = (at.row.unit0 + at.unit + u) * UNIT + (lane >> 2);
                    const int end = min(at.row.end, (at.row.unit0 + at.unit + at.n) * UNIT);
                    float *to = a.logits + (((int64_t)at.r * a.kv_heads + kv_head) * a.positions + key) * a.group + h;
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int more = 16 * g + 8 * (j >> 1);
                            if (key + more >= at.row.first && key + more < end && h + (j & 1) < a.group) to[more * a.group + (j & 1)] = x[g][j] * unscale[t][j & 1];
                        }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(fmaxf(x[0][j], x[0][j + 2]), fmaxf(x[1][j], x[1][j + 2]));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                    const float c = unscale[t][j];
                    top = fmaxf(top * c, m[t][j]);
                    const float from = top == -INFINITY ? 0.f : -top;  // (keys of bad pages only, so far)
                    shrink[t][j] = power2(m[t][j] + from);
                    m[t][j] = top;
                    float sum = 0.f;
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int i = j; i < 4; i += 2) {
                            x[g][i] = power2(fmaf(x[g][i], c, from)) * P::UP;
                            sum += x[g][i];
                        }
                    l[t][j] = l[t][j] * shrink[t][j] + sum;
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t w0[P::N], w1[P::N];
                    P::split(x[g][0], x[g][1], w0);
                    P::split(x[g][2], x[g][3], w1);
#pragma unroll
                    for (int j = 0; j < P::N; ++j) p[t][g][j][0] = transposed(w0[j]), p[t][g][j][1] = transposed(w1[j]);
                }
            }

            tile = next_tile(true);
            // The tensor cores cut a sum's last bits off instead of rounding: they add up one step, the sum over steps is rounded.  The small
            // parts go first.  Four tiles of 16 elements at a time, so that four sums are in the making.
            constexpr int BATCH = NT == 1 && W <= 8 ? 4 : 2;
#pragma unroll
            for (int s0 = 0; s0 < DP / 16; s0 += BATCH) {
                float d[BATCH][NT][4];
                uint32_t v[BATCH][2][4];
                if constexpr (E4M3) {
#pragma unroll
                    for (int s = 0; s < BATCH; s += 2)
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            uint32_t r[4];
                            ldmatrix4_trans(r, ((tile + v_place) ^ ((s0 + s) * 16)) + UNIT * g * S::ROW);
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                // rows of the product: elements 2i, then 2i + 1, of the 16
                                halves_of_e4m3(__byte_perm(r[k], 0, 0x3120), v[s + k][g][0], v[s + k][g][1]);
                                halves_of_e4m3(__byte_perm(r[k + 2], 0, 0x3120), v[s + k][g][2], v[s + k][g][3]);
                            }
                        }
                } else {
#pragma unroll
                    for (int s = 0; s < BATCH; ++s)
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                            ldmatrix4_trans(v[s][g], ((tile + v_place) ^ ((s0 + s) * 32)) + UNIT * g * S::ROW);
                }
#pragma unroll
                for (int j = P::N - 1; j >= 0; --j)
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int s = 0; s < BATCH; ++s)
#pragma unroll
                            for (int t = 0; t < NT; ++t) P::mma(d[s][t], v[s][g], p[t][g][j], j == P::N - 1 && g == 0);
#pragma unroll
                for (int s = 0; s < BATCH; ++s)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[t][s0 + s][j] = o[t][s0 + s][j] * shrink[t][j & 1] + d[s][t][j];
            }
        }

        // the next piece; its queries are asked for while this one is put away
        const int row = at.r, phase = at.phase;
        const bool whole = !apart && at.unit == 0 && at.n == at.row.units;
        next_piece(at);
        if (S::EARLY_QUERIES && at.phase != DONE) ask_queries();

        // into shared memory, by heads: where the ring was, if this was the last piece
        float *result = reinterpret_cast<float *>(phase == LAST ? my_ring : results + warp * S::RESULT);
        float2 *stats = reinterpret_cast<float2 *>(result + S::HEADS * DP);
        __syncwarp();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 4);
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 8);
                l[t][j] += __shfl_xor_sync(0xFFFFFFFFu, l[t][j], 16);
                if (lane < 4) stats[8 * t + 2 * lane + j] = make_float2(m[t][j], l[t][j]);
            }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = 16 * s + (E4M3 ? 2 * (lane >> 2) + (j >> 1) : (lane >> 2) + 8 * (j >> 1));
                    result[result_at<DP>(8 * t + 2 * (lane & 3) + (j & 1), d)] = o[t][s][j];
                }
        __syncwarp();
        if (whole) {  // nobody else has any of it
#pragma unroll 1
            for (int h = 0; h < heads; ++h) {
                const float f = inverse_sum(stats[h].y) * a.v_scale;
#pragma unroll 1
                for (int d0 = 0; d0 < DP; d0 += 128) {
                    const int d = d0 + 4 * lane;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (d < a.dim) {
                        v = *reinterpret_cast<const float4 *>(result + result_at<DP>(h, d));
                        v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
                    }
                    write_output(a, row, head0, h * a.dim + d, v, d < a.dim);
                }
            }
            if (WEIGHTS && lane < heads) a.norms[(int64_t)row * a.q_heads + head0 + lane] = norm_of(stats[lane].x, inverse_sum(stats[lane].y) * P::UP);
            __syncwarp();
            if (phase != MIDDLE && lane == 0) mine[phase == FIRST ? 0 : 1].n = 0;
        }
    }
    __syncthreads();

    // ---- what the warps have of the same segment, together ----
    // Entry 2w is warp w's first piece, 2w + 1 its last: in the order of the units.
    const Entry entry = entries[lane < 2 * W ? lane : 0];
    const bool exists = lane < 2 * W && entry.n > 0;
    const uint32_t there = __ballot_sync(0xFFFFFFFFu, exists);
    const uint32_t lower = there & ((1u << lane) - 1);
    const int previous = lower ? 31 - __clz(lower) : 0;
    const int previous_row = __shfl_sync(0xFFFFFFFFu, entry.row, previous), previous_segment = __shfl_sync(0xFFFFFFFFu, entry.segment, previous);
    uint32_t starts = __ballot_sync(0xFFFFFFFFu, exists && (lower == 0 || previous_row != entry.row || previous_segment != entry.segment));
    const auto result_of = [&](int i) {
        return reinterpret_cast<const float *>(i & 1 ? smem + (i >> 1) * S::SLOTS * S::TILE : results + (i >> 1) * S::RESULT);
    };
    const auto members_of = [&](int i0) {  // the entries of the segment that begins with entry i0
        const uint32_t from = ~((1u << i0) - 1), behind = starts & from & (from << 1);
        return there & from & (behind ? (1u << (__ffs(behind) - 1)) - 1 : 0xFFFFFFFFu);
    };
    float *factors = reinterpret_cast<float *>(smem + S::RESULT);                    // [entry][head]: of its result
    float2 *sums = reinterpret_cast<float2 *>(factors + 2 * W * S::HEADS);           // [first entry][head]: largest logit, sum of weights
    {
        const int i = threadIdx.x / S::HEADS, h = threadIdx.x % S::HEADS;
        if (i < 2 * W && (there >> i & 1u)) {
            const int i0 = 31 - __clz(starts & ((2u << i) - 1));
            const uint32_t members = members_of(i0);
            const auto stat = [&](uint32_t b) { return reinterpret_cast<const float2 *>(result_of(__ffs(b) - 1) + S::HEADS * DP)[h]; };
            const float own_top = stat(1u << i).x;
            float top = -INFINITY, sum = 0.f;
#pragma unroll 1
            for (uint32_t b = members; b != 0; b &= b - 1) top = fmaxf(top, stat(b).x);
            const float from = top == -INFINITY ? 0.f : top;
#pragma unroll 1
            for (uint32_t b = members; b != 0; b &= b - 1) sum += stat(b).y * power2(stat(b).x - from);
            factors[threadIdx.x] = power2(own_top - from);
            if (i == i0) sums[threadIdx.x] = make_float2(top, sum);
        }
    }
    __syncthreads();
    // a block has at most one segment that began before it and one that goes on behind it (or one that does both)
    int n_unfinished = 0, unfinished0 = 0, unfinished1 = 0;  // those segments' first entries
    int turn = warp;                                         // the warp's next head: the segments' heads go round
#pragma unroll 1
    for (uint32_t left = starts; left != 0; left &= left - 1) {
        const int i0 = __ffs(left) - 1;
        const uint32_t members = members_of(i0);
        const Entry &f = entries[i0], &g = entries[31 - __clz(members)];
        const bool whole = f.unit == 0 && g.unit + g.n == g.units;
        if (!whole) {
            if (n_unfinished++ == 0) unfinished0 = i0;
            else unfinished1 = i0;
        }
        const int kv_head = a.tiles == 1 ? f.segment : f.segment / a.tiles, tile = f.segment - kv_head * a.tiles;
        const int head0 = kv_head * a.group + tile * S::HEADS, heads = min(S::HEADS, a.group - tile * S::HEADS);
        float *part = a.parts + (int64_t)(2 * blockIdx.x + (f.unit == 0 ? 1 : 0)) * S::PART;
#pragma unroll 1
        for (; turn < heads; turn += W) {  // a warp a head
            const int h = turn;
            const float2 st = sums[i0 * S::HEADS + h];
            const float inv = inverse_sum(st.y), w = whole ? inv * a.v_scale : 1.f;
#pragma unroll 1
            for (int d0 = 0; d0 < DP; d0 += 128) {
                const int d = d0 + 4 * lane;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (d < a.dim) {
#pragma unroll 1
                    for (uint32_t b = members; b != 0;) {  // four at a time
                        float c[4];
                        float4 x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int i = b != 0 ? __ffs(b) - 1 : i0;
                            c[k] = b != 0 ? factors[i * S::HEADS + h] : 0.f;
                            x[k] = *reinterpret_cast<const float4 *>(result_of(i) + result_at<DP>(h, d));
                            if (b == 0) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            b &= b - 1;
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) v = make_float4(v.x + c[k] * x[k].x, v.y + c[k] * x[k].y, v.z + c[k] * x[k].z, v.w + c[k] * x[k].w);
                    }
                    v = make_float4(v.x * w, v.y * w, v.z * w, v.w * w);
                    if (!whole) __stcg(reinterpret_cast<float4 *>(part + h * DP + d), v);
                }
                if (whole) write_output(a, f.row, head0, h * a.dim + d, v, d < a.dim);
            }
            if (lane == 0 && !whole) __stcg(reinterpret_cast<float2 *>(part + S::HEADS * DP) + h, st);
            if (WEIGHTS && lane == 0 && whole) a.norms[(int64_t)f.row * a.q_heads + head0 + h] = norm_of(st.x, inv * P::UP);
        }
        turn -= heads;
    }

    if (n_unfinished > 0) {
        int *part_first = is_last + 2, *part_count = is_last + 4;  // of the two segments: the first of their blocks, and how many
        __syncthreads();  // all of the parts is written
        if ((int)threadIdx.x < n_unfinished) {
            const Entry &f = entries[threadIdx.x == 0 ? unfinished0 : unfinished1];
            int first = first_block, n_parts = parts_apart, before;
            if (!apart) {
                const uint32_t start = u0 + f.start + BEGIN;  // of its units
                first = start / per_block;
                n_parts = (start + f.units - 1) / per_block - first + 1;
            }
            part_first[threadIdx.x] = first, part_count[threadIdx.x] = n_parts;
            // Where segments are many they go by the block that they begin in: of those that go on behind it a block has one.  So the counters
            // are as many as blocks at most, and lie in the same place for calls of any size.
            int *counter = a.counters + ((int64_t)a.rows * segments_row <= gridDim.x ? f.row * segments_row + f.segment : first);
            asm volatile("fence.acq_rel.gpu;\n\tatom.acq_rel.gpu.global.add.s32 %0, [%1], 1;\n\tfence.acq_rel.gpu;" : "=r"(before) : "l"(counter) : "memory");
            if (before == n_parts - 1) *counter = 0;  // for the next call
            is_last[threadIdx.x] = before == n_parts - 1;
        }
        __syncthreads();
        // a warp a head of one of the two, a lane the weight of a part
        const int each = min(S::HEADS, a.group);
#pragma unroll 1
        for (int turn = warp; turn < n_unfinished * each; turn += W) {
            const int k = turn >= each, h = turn - k * each;
            if (!is_last[k]) continue;
            const Entry &f = entries[k == 0 ? unfinished0 : unfinished1];
            const int kv_head = a.tiles == 1 ? f.segment : f.segment / a.tiles, tile = f.segment - kv_head * a.tiles;
            const int head0 = kv_head * a.group + tile * S::HEADS, heads = min(S::HEADS, a.group - tile * S::HEADS);
            if (h >= heads) continue;
            const int first = part_first[k], n_parts = part_count[k];
            // a block's part that begins a segment has a place of its own: the block may also have the end of the one before
            const auto part_of = [&](int i) { return a.parts + (2 * (first + i) + (i == 0 ? 1 : 0)) * S::PART; };
            const auto stat_of = [&](int i) { return __ldcg(reinterpret_cast<const float2 *>(part_of(i) + S::HEADS * DP) + h); };
            constexpr int ACROSS = (DP + 127) / 128;
            const auto sums_of = [&](int i, int c) {
                const int d = 128 * c + 4 * lane;
                return d < a.dim ? __ldcg(reinterpret_cast<const float4 *>(part_of(i) + h * DP + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            constexpr int EARLY = 8;  // parts whose sums are on their way while the weights are made
            float4 early[EARLY][ACROSS];
            float2 st = lane < n_parts ? stat_of(lane) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int n = 0; n < EARLY; ++n)
#pragma unroll
                for (int c = 0; c < ACROSS; ++c) early[n][c] = sums_of(min(n, n_parts - 1), c);
            float top = st.x;
#pragma unroll 1
            for (int n = lane + 32; n < n_parts; n += 32) top = fmaxf(top, stat_of(n).x);
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, i));
            const float from = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float4 v[ACROSS];
#pragma unroll
            for (int c = 0; c < ACROSS; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            const auto add = [&](const float4 &x, float w, int c) {
                v[c] = make_float4(v[c].x + w * x.x, v[c].y + w * x.y, v[c].z + w * x.z, v[c].w + w * x.w);
            };
#pragma unroll 1
            for (int n0 = 0; n0 < n_parts; n0 += 32) {
                if (n0 > 0) st = n0 + lane < n_parts ? stat_of(n0 + lane) : make_float2(-INFINITY, 0.f);
                const float weight = power2(st.x - from);  // (of a part that is not there: 0)
                sum += weight * st.y;
                int n = 0;
                if (n0 == 0) {
#pragma unroll
                    for (; n < EARLY; ++n) {
                        const float w = __shfl_sync(0xFFFFFFFFu, weight, n);
#pragma unroll
                        for (int c = 0; c < ACROSS; ++c)
                            if (n < n_parts) add(early[n][c], w, c);
                    }
                }
                const int n1 = min(32, n_parts - n0);
                // eight parts at a time, the last ones with the weight 0
#pragma unroll 1
                for (; n < n1; n += 8) {
                    float4 x[8][ACROSS];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int c = 0; c < ACROSS; ++c) x[i][c] = sums_of(n0 + min(n + i, n1 - 1), c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float w = n + i < n1 ? __shfl_sync(0xFFFFFFFFu, weight, (n + i) & 31) : 0.f;
#pragma unroll
                        for (int c = 0; c < ACROSS; ++c)
                            if (n + i < n1) add(x[i][c], w, c);
                    }
                }
            }
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, i);
            const float inv = inverse_sum(sum), w = inv * a.v_scale;
#pragma unroll
            for (int c = 0; c < ACROSS; ++c) {
                const int d = 128 * c + 4 * lane;
                write_output(a, f.row, head0, h * a.dim + d, make_float4(v[c].x * w, v[c].y * w, v[c].z * w, v[c].w * w), d < a.dim);
            }
            if (WEIGHTS && lane == 0) a.norms[(int64_t)f.row * a.q_heads + head0 + h] = norm_of(top, inv * P::UP);
        }
    }

    // rows that see nothing get their zeros
#pragma unroll 1
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const Row x = row_of(a, r);
        if (x.seq < 0 || x.units > 0) continue;
        const int n4 = a.q_heads * a.dim / 4;
#pragma unroll 1
        for (int e = threadIdx.x; e < (n4 + 31) / 32 * 32; e += S::THREADS)
            write_output(a, r, 0, 4 * e, make_float4(0.f, 0.f, 0.f, 0.f), e < n4);
    }
}

// Adds to every seen token's weight what its query heads gave it.  The logits of the attention kernel are read once: a thread has one token's,
// four heads at a time where they are aligned.
__global__ void __launch_bounds__(256) attention_weights_kernel(const AttnArgs a, float *weights, int64_t weights_stride, int64_t weights_len) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.z, kv_head = blockIdx.y;
    const Row r = row_of(a, row);
    const float2 *norms = a.norms + (int64_t)row * a.q_heads + kv_head * a.group;
    const int64_t end = min((int64_t)r.end, weights_len);
    const int64_t segment = (int64_t)row * a.kv_heads + kv_head;
    for (int64_t key = r.first + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; key < end; key += (int64_t)gridDim.x * blockDim.x) {
        const float *s = a.logits + (segment * a.positions + key) * a.group;
        float *to = weights + segment * weights_stride + key;
        const float before = *to;
        float given = 0.f;
        if (a.group % 4 == 0) {
#pragma unroll 4
            for (int h = 0; h < a.group; h += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(s + h);
                given += power2(x.x - norms[h].x) * norms[h].y + power2(x.y - norms[h + 1].x) * norms[h + 1].y;
                given += power2(x.z - norms[h + 2].x) * norms[h + 2].y + power2(x.w - norms[h + 3].x) * norms[h + 3].y;
            }
        } else {
#pragma unroll 8
            for (int h = 0; h < a.group; ++h) given += power2(s[h] - norms[h].x) * norms[h].y;
        }
        *to = before + given;
    }
}

// More than eight query heads to a key head: sixteen in one pass over the keys, where the registers hold them.
bool takes_16_heads(int64_t group, int64_t dim) { return group > 8 && dim <= 128; }

int check_heads(int64_t rows, int64_t q_heads, const jq_kv_cache *c) {
    if (rows < 0 || q_heads <= 0) return set_error(JQ_ERR_INVALID_ARG, "attention: a size is not positive");
    if (q_heads % c->num_kv_heads != 0)
        return set_error(JQ_ERR_SHAPE, "attention: %lld query heads do not divide among %lld key heads", (long long)q_heads, (long long)c->num_kv_heads);
    if (rows > 0x7FFFFFF || q_heads > 65535) return set_error(JQ_ERR_TOO_LARGE, "attention: too many rows or heads");
    // the kernel counts units in 32 bits, with BEGIN more for every segment; and nothing that follows from these sizes overflows
    const int64_t group = q_heads / c->num_kv_heads, heads = takes_16_heads(group, c->head_dim) ? 16 : 8;
    const double units = (double)rows * (double)c->num_kv_heads * (double)((group + heads - 1) / heads) * (double)((c->max_pages * c->page_size + UNIT - 1) / UNIT);
    if (units > 536870912.0)
        return set_error(JQ_ERR_TOO_LARGE, "attention: %lld rows of %lld key heads with room for %lld tokens are more than 2^29 units of %d", (long long)rows,
                         (long long)c->num_kv_heads, (long long)(c->max_pages * c->page_size), UNIT);
    return JQ_OK;
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

struct Workspace {
    size_t parts, norms, logits, total;
};
int workspace_of(int64_t rows, int64_t q_heads, const jq_kv_cache *c, bool weights, Workspace *w) {
    DeviceCaps caps;
    if (int rc = device_caps(&caps)) return rc;
    w->parts = rounded(sizeof(int) * (size_t)caps.sm_count);  // behind the counters, of which there is one for a block at most
    const int64_t dim = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256, heads = takes_16_heads(q_heads / c->num_kv_heads, c->head_dim) ? 16 : 8;
    const size_t part = heads * dim + 2 * heads;  // floats: Shape::PART of the instance that launch_for() takes
    w->norms = w->parts + rounded(2 * (size_t)caps.sm_count * part * sizeof(float));
    w->logits = w->norms + (weights ? rounded(sizeof(float2) * (size_t)rows * q_heads) : 0);
    w->total = w->logits + (weights ? rounded(sizeof(float) * (size_t)rows * q_heads * (size_t)(c->max_pages * c->page_size)) : 0);
    if (w->total < JQ_PAGED_ATTENTION_COUNTERS(rows, q_heads)) w->total = rounded(JQ_PAGED_ATTENTION_COUNTERS(rows, q_heads));  // (which the caller zeroes)
    return JQ_OK;
}

template <typename T, int DP, int NT, bool WEIGHTS>
int launch_as(cudaStream_t st, AttnArgs &a, int sm_count) {
    using S = Shape<T, DP, NT>;
    const auto kernel = paged_attention_kernel<T, DP, NT, WEIGHTS>;
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), S::SMEM, true)) return rc;
    a.tiles = (a.group + S::HEADS - 1) / S::HEADS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sm_count);
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
int launch_for(cudaStream_t st, AttnArgs &a, int sm_count) {
    if (a.dim > 128) return launch_as<T, 256, 1, WEIGHTS>(st, a, sm_count);
    if (takes_16_heads(a.group, a.dim)) return a.dim > 64 ? launch_as<T, 128, 2, WEIGHTS>(st, a, sm_count) : launch_as<T, 64, 2, WEIGHTS>(st, a, sm_count);
    return a.dim > 64 ? launch_as<T, 128, 1, WEIGHTS>(st, a, sm_count) : launch_as<T, 64, 1, WEIGHTS>(st, a, sm_count);
}

template <bool WEIGHTS>
int launch_type(cudaStream_t st, AttnArgs &a, int type, int sm_count) {
    if (type == JQ_KV_F16) return launch_for<KvF16, WEIGHTS>(st, a, sm_count);
    if (type == JQ_KV_BF16) return launch_for<KvBf16, WEIGHTS>(st, a, sm_count);
    return launch_for<KvE4m3, WEIGHTS>(st, a, sm_count);
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
    if (num_rows == 0) return JQ_OK;  // (before the outputs: an empty tensor has no address)
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
    a.q = d_q, a.q_row = q_stride_row, a.q_head = q_stride_head;
    a.k = static_cast<const char *>(cache->d_k), a.v = static_cast<const char *>(cache->d_v);
    a.lens = d_lens, a.seqs = d_seqs, a.out = d_out, a.xq = static_cast<uint8_t *>(d_xq);
    a.scale = 2.f * (float)std::frexp((double)scale * cache->k_scale * 1.4426950408889634, &a.scale_exponent);
    a.scale_exponent -= 1;
    a.v_scale = cache->v_scale;
    a.rows = (int)num_rows, a.q_heads = (int)num_q_heads, a.kv_heads = (int)cache->num_kv_heads, a.group = a.q_heads / a.kv_heads, a.dim = (int)dim;
    a.positions = (int)(cache->max_pages * cache->page_size);
    a.grouped = cache->page_size % UNIT == 0;
    a.window = window >= a.positions ? 0 : (int)window;
    a.n_super = (int)(num_q_heads * dim / SUPER), a.order = order, a.s_mode = s_mode;
    char *ws = static_cast<char *>(d_ws);
    a.counters = reinterpret_cast<int *>(ws);
    a.parts = reinterpret_cast<float *>(ws + w.parts);
    a.norms = reinterpret_cast<float2 *>(ws + w.norms);
    a.logits = reinterpret_cast<float *>(ws + w.logits);
    a.fault = device_fault_ptr();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d_weights == nullptr) return launch_type<false>(st, a, cache->type, caps.sm_count);
    if (int rc = launch_type<true>(st, a, cache->type, caps.sm_count)) return rc;
    if (a.positions == 0) return JQ_OK;
    // (blocks for eight per SM over all rows and heads at least, as far as there are tokens; they walk on where sequences are longer)
    const int64_t segments = num_rows * a.kv_heads, most = (8 * (int64_t)caps.sm_count + segments - 1) / segments;
    int64_t across = (a.positions + 255) / 256;
    if (across > 16 && across > most) across = most > 16 ? most : 16;
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
