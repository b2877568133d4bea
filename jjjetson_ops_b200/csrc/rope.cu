// Rotary positions: a pair (a, b) of a head turns by position * frequency, (a cos - b sin, b cos + a sin).  Two entry points share one
// kernel: heads in, heads out, and the fused projection's rows, whose keys and values go on into the pages of a cache.
//
// What bounds it: bytes (8 per element of a query, 6 per element of a key or value).  Everything else is done once for a row: the angles
// and the row's place in the cache, by the block together, into shared memory.  A thread keeps one group of pairs (its sines and
// cosines in registers) and walks over the heads.
#include "kv_cache.cuh"

#include <cmath>

namespace jq {

namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_ROWS = 2;     // of a block

struct RopeArgs {
    const float *x;
    int64_t x_row, x_head;
    float *out;
    int64_t out_row, out_head;
    const int32_t *positions;
    const unsigned long long *table;
    int rows, rows_per_block;
    int heads;    // that are rotated into `out`
    int kv_heads; // then so many of keys and of values
    int units;    // groups of 2 * W elements that a block takes of a head
    int all_units;    // that a head has: more where it is wider than a block (WIDE)
    int rotary_units;
    int half;     // rotary_dim / 2
    int heads_per_block_y;  // heads (of all kinds) that a block of this launch takes
    int dim;
    float mscale;
    // the cache
    KvIndex ix;
    void *k, *v;
    const int32_t *index, *seqs;
    float k_scale, v_scale;
    int *fault;
};

template <int N>
__device__ __forceinline__ void load_floats(float *to, const float *from) {
    if constexpr (N == 1) to[0] = from[0];
    if constexpr (N == 2) {
        const float2 v = *reinterpret_cast<const float2 *>(from);
        to[0] = v.x, to[1] = v.y;
    }
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(from + i);
            to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void store_floats(float *to, const float *from) {
    if constexpr (N == 1) to[0] = from[0];
    if constexpr (N == 2) *reinterpret_cast<float2 *>(to) = make_float2(from[0], from[1]);
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(to + i) = make_float4(from[i], from[i + 1], from[i + 2], from[i + 3]);
    }
}

// (spelled out: every instance gives the same bits, whatever strides and alignment it was chosen for)
__device__ __forceinline__ float turned_first(float a, float b, float c, float s) { return __fmaf_rn(a, c, -__fmul_rn(b, s)); }
__device__ __forceinline__ float turned_second(float a, float b, float c, float s) { return __fmaf_rn(b, c, __fmul_rn(a, s)); }

// One group of W pairs: where its two parts lie in a head.
struct Unit {
    int first, second;  // offsets of the first and the second elements of the pairs (half layout) or of the halves of 2 W in a row
    bool turns;
};

// W: pairs per thread and head (4, 2 or 1, by divisibility and alignment).  T: the cache's element type; void: no cache.  WIDE: heads of more
// pairs than a block has threads, shared by blocks next to one another (an instance of its own: in all of them the index more cost
// 10.4 -> 10.9 us for 2049 rows of 25 x 80).
template <int W, bool INTERLEAVED, typename T, bool WIDE>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeArgs a) {
    constexpr bool CACHE = !std::is_same<T, void>::value;
    extern __shared__ __align__(16) float2 turn[];  // [rows_per_block][half]: cosine and sine
    __shared__ int64_t place[ROPE_MAX_ROWS];        // element offset of the row's token in the cache, -1: none
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row0 = blockIdx.x * a.rows_per_block;
    const int rows = min(a.rows_per_block, a.rows - row0);
    const int all_heads = a.heads + (CACHE ? 2 * a.kv_heads : 0);
    const int u = threadIdx.x % a.units + (WIDE ? blockIdx.z * a.units : 0), lane_head = threadIdx.x / a.units, step = blockDim.x / a.units;
    const int head0 = blockIdx.y * a.heads_per_block_y, head1 = WIDE && u >= a.all_units ? head0 : min(all_heads, head0 + a.heads_per_block_y);
    Unit at;
    at.turns = u < a.rotary_units;
    at.first = INTERLEAVED || !at.turns ? 2 * W * u : W * u;
    at.second = INTERLEAVED || !at.turns ? at.first + W : a.half + W * u;

    // a head's elements are asked for while the one before it is worked on; the first one's while the angles are computed
    float next_p[W], next_q[W];
    int next_row = 0, next_head = head0 + lane_head;
    const float *next_x = a.x + (int64_t)row0 * a.x_row + (int64_t)next_head * a.x_head;
    const auto load = [&]() {
        if (INTERLEAVED && W >= 2) {
            float y[2 * W];
            load_floats<2 * W>(y, next_x + at.first);
#pragma unroll
            for (int i = 0; i < W; ++i) next_p[i] = y[i], next_q[i] = y[W + i];
        } else {
            load_floats<W>(next_p, next_x + at.first);
            load_floats<W>(next_q, next_x + at.second);
        }
        next_head += step;
        next_x += step * a.x_head;
        if (next_head >= head1) {
            ++next_row;
            next_head = head0 + lane_head;
            next_x = a.x + (int64_t)(row0 + next_row) * a.x_row + (int64_t)next_head * a.x_head;
        }
    };
    if (next_head < head1) load();

    for (int i = threadIdx.x; CACHE && head1 > a.heads && i < rows; i += blockDim.x) {
        const int row = row0 + i;
        const int32_t seq = a.seqs != nullptr ? a.seqs[row] : row, token = a.index[row];
        int64_t to = -1;
        if (seq >= 0 && seq < a.ix.num_seqs && token >= 0 && token < (int64_t)a.ix.max_pages * a.ix.page_size) {
            to = kv_offset(a.ix, (uint32_t)token, a.ix.table[(int64_t)seq * a.ix.table_stride + kv_page_of(a.ix, (uint32_t)token)]);
            if (to < 0) report_bad_page(a.fault);
        }
        place[i] = to;
    }
    for (int i = threadIdx.x; i < rows * a.half; i += blockDim.x) {
        const int row = i / a.half, pair = i - row * a.half;
        float s, c;
        uint32_t quarters;
        sincospif(rope_half_turns(a.table[pair], a.positions[row0 + row], &quarters), &s, &c);
        rope_add_quarters(quarters, &c, &s);
        turn[i] = make_float2(c * a.mscale, s * a.mscale);
    }
    __syncthreads();

    for (int row = 0; row < rows; ++row) {
        float c[W], s[W];
        if (at.turns) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float2 t = turn[row * a.half + W * u + i];
                c[i] = t.x, s[i] = t.y;
            }
        }
        for (int head = head0 + lane_head; head < head1; head += step) {
            float p[W], q[W];
#pragma unroll
            for (int i = 0; i < W; ++i) p[i] = next_p[i], q[i] = next_q[i];
            if (next_row < rows) load();
            const bool is_value = CACHE && head >= a.heads + a.kv_heads;
            if (at.turns && !is_value) {
                float y[2 * W];
                if (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < W; ++i) y[i] = p[i], y[W + i] = q[i];
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float e = y[2 * i], o = y[2 * i + 1];
                        y[2 * i] = turned_first(e, o, c[i], s[i]);
                        y[2 * i + 1] = turned_second(e, o, c[i], s[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        y[i] = turned_first(p[i], q[i], c[i], s[i]);
                        y[W + i] = turned_second(p[i], q[i], c[i], s[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < W; ++i) p[i] = y[i], q[i] = y[W + i];
            }
            if (!CACHE || head < a.heads) {
                float *y = a.out + (int64_t)(row0 + row) * a.out_row + (int64_t)head * a.out_head;
                if (INTERLEAVED && W >= 2) {
                    float both[2 * W];
#pragma unroll
                    for (int i = 0; i < W; ++i) both[i] = p[i], both[W + i] = q[i];
                    store_floats<2 * W>(y + at.first, both);
                } else {
                    store_floats<W>(y + at.first, p);
                    store_floats<W>(y + at.second, q);
                }
            }
            if constexpr (CACHE) {
                if (head >= a.heads && place[row] >= 0) {
                    using E = typename T::Element;
                    const int h = head - a.heads - (is_value ? a.kv_heads : 0);
                    E *to = static_cast<E *>(is_value ? a.v : a.k) + place[row] + (int64_t)h * a.ix.stride_head;
                    const float scale = is_value ? a.v_scale : a.k_scale;
                    if (scale != 1.f) {
#pragma unroll
                        for (int i = 0; i < W; ++i) p[i] = __fdiv_rn(p[i], scale), q[i] = __fdiv_rn(q[i], scale);
                    }
                    if (at.second == at.first + W) {
                        float y[2 * W];
#pragma unroll
                        for (int i = 0; i < W; ++i) y[i] = p[i], y[W + i] = q[i];
                        store_elements<T, 2 * W>(to + at.first, y);
                    } else if constexpr (W >= 2) {
                        store_elements<T, W>(to + at.first, p);
                        store_elements<T, W>(to + at.second, q);
                    } else {
                        const uint32_t both = pack2(T{}, p[0], q[0]);
                        if constexpr (sizeof(E) == 2) {
                            reinterpret_cast<uint16_t *>(to)[at.first] = (uint16_t)both;
                            reinterpret_cast<uint16_t *>(to)[at.second] = (uint16_t)(both >> 16);
                        } else {
                            reinterpret_cast<uint8_t *>(to)[at.first] = (uint8_t)both;
                            reinterpret_cast<uint8_t *>(to)[at.second] = (uint8_t)(both >> 8);
                        }
                    }
                }
            }
        }
    }
}

// Pairs per thread: the most for which the rotated and the other elements of a head divide and all addresses are aligned.
int pairs_per_thread(const RopeArgs &a, int rotary_dim, int interleaved) {
    for (int w = 4; w > 1; w >>= 1) {
        if (rotary_dim % (2 * w) != 0 || (a.dim - rotary_dim) % (2 * w) != 0) continue;
        const uintptr_t mask = (w == 4 || interleaved ? 16 : 8) - 1;
        const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)(a.x_row * 4) | (uintptr_t)(a.x_head * 4) |
                               (uintptr_t)(a.out_row * 4) | (uintptr_t)(a.out_head * 4);
        if ((bits & mask) != 0) continue;
        return w;
    }
    return 1;
}

template <int W, bool INTERLEAVED, typename T, bool WIDE = false>
int launch_rope_as(cudaStream_t st, RopeArgs &a, int rotary_dim) {
    DeviceCaps caps;
    if (int rc = device_caps(&caps)) return rc;
    a.all_units = a.dim / (2 * W);
    a.rotary_units = rotary_dim / (2 * W);
    if constexpr (W == 1 && std::is_same<T, void>::value && !WIDE) {  // (a cache's heads have 128 pairs at most)
        if (a.all_units > ROPE_THREADS) return launch_rope_as<W, INTERLEAVED, T, true>(st, a, rotary_dim);
    }
    const int across = (a.all_units + ROPE_THREADS - 1) / ROPE_THREADS;
    a.units = (a.all_units + across - 1) / across;
    const int all_heads = a.heads + 2 * a.kv_heads, at_once = ROPE_THREADS / a.units;
    const int used = at_once < all_heads ? at_once : all_heads;
    // Few rows: a block per row and as many heads as it takes at once.  Many: a block takes some rows, and all their heads.
    const int64_t blocks_per_row = (all_heads + used - 1) / used;
    const bool few = a.rows * blocks_per_row <= 4 * (int64_t)caps.sm_count;
    // (two rows where that leaves every SM its eight blocks.  us with four rows, two, one: 8192 rows of 64 x 128 85.4, 83.7, 84.0; 4097 rows
    // of 32 + 2 x 8 heads into a cache 34.4, 31.4, 33.3; 2049 of 25 x 80 10.2, 9.4, 9.1)
    a.rows_per_block = few || a.rows < ROPE_MAX_ROWS * 8 * (int64_t)caps.sm_count ? 1 : ROPE_MAX_ROWS;
    a.heads_per_block_y = few ? used : all_heads;
    const size_t smem = sizeof(float2) * (size_t)a.rows_per_block * a.half;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block),
                       (unsigned)((all_heads + a.heads_per_block_y - 1) / a.heads_per_block_y), (unsigned)across);
    cfg.blockDim = dim3((unsigned)(used * a.units));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    JQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_kernel<W, INTERLEAVED, T, WIDE>, (const RopeArgs)a));
    return JQ_OK;
}

template <typename T>
int launch_rope(cudaStream_t st, RopeArgs &a, int rotary_dim, int interleaved) {
    const int w = pairs_per_thread(a, rotary_dim, interleaved);
    if (interleaved) {
        if (w == 4) return launch_rope_as<4, true, T>(st, a, rotary_dim);
        if (w == 2) return launch_rope_as<2, true, T>(st, a, rotary_dim);
        return launch_rope_as<1, true, T>(st, a, rotary_dim);
    }
    if (w == 4) return launch_rope_as<4, false, T>(st, a, rotary_dim);
    if (w == 2) return launch_rope_as<2, false, T>(st, a, rotary_dim);
    return launch_rope_as<1, false, T>(st, a, rotary_dim);
}

int check_rope(int64_t rows, int64_t heads, int64_t dim, int64_t rotary_dim, float mscale) {
    if (rows < 0 || heads < 0 || dim <= 0) return set_error(JQ_ERR_INVALID_ARG, "rope: negative size");
    if (dim % 2 != 0 || dim > 1024) return set_error(JQ_ERR_SHAPE, "rope: head_dim = %lld is not even or above 1024", (long long)dim);
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > dim)
        return set_error(JQ_ERR_SHAPE, "rope: rotary_dim = %lld is not an even number up to head_dim = %lld", (long long)rotary_dim, (long long)dim);
    if (rows > 0x7FFFFFF0 || heads > 65535) return set_error(JQ_ERR_TOO_LARGE, "rope: too many rows or heads");
    if (!std::isfinite(mscale)) return set_error(JQ_ERR_INVALID_ARG, "rope: mscale is not finite");
    return JQ_OK;
}

// In the 64 bits of a long double: 53 are a step of 2^-56 turns for a fast pair, which 2^31 positions make 2^-25 turns of.
uint64_t steps_of(long double radians) {
    constexpr long double TWO_PI = 6.283185307179586476925286766559L;
    long double turns = radians / TWO_PI;
    turns -= floorl(turns);  // whole turns do not count
    const long double steps = floorl(turns * 18446744073709551616.0L + 0.5L);
    return steps >= 18446744073709551616.0L ? 0 : (uint64_t)steps;
}

}  // namespace

int check_kv_cache(const jq_kv_cache *c, KvIndex *ix) {
    if (c == nullptr) return set_error(JQ_ERR_INVALID_ARG, "kv cache: null pointer");
    if (c->type != JQ_KV_F16 && c->type != JQ_KV_BF16 && c->type != JQ_KV_E4M3)
        return set_error(JQ_ERR_INVALID_ARG, "kv cache: unknown type %d", c->type);
    if (c->num_pages <= 0 || c->page_size <= 0 || c->num_kv_heads <= 0 || c->num_seqs < 0 || c->max_pages < 0)
        return set_error(JQ_ERR_INVALID_ARG, "kv cache: a size is not positive");
    if (c->head_dim <= 0 || c->head_dim % 16 != 0 || c->head_dim > KV_MAX_DIM)
        return set_error(JQ_ERR_SHAPE, "kv cache: head_dim = %lld is not a multiple of 16 up to %lld", (long long)c->head_dim, (long long)KV_MAX_DIM);
    if (c->num_pages > 0x7FFFFFFF || c->page_size > 0x7FFFFFFF || c->num_kv_heads > 65535 || c->num_seqs > 0x7FFFFFFF ||
        c->max_pages > 0x7FFFFFFF || (c->max_pages > 0 && c->page_size > 0x7FFFFF00 / c->max_pages))
        return set_error(JQ_ERR_TOO_LARGE, "kv cache: more than 2^31 tokens in a sequence, or pages, or sequences");
    if (c->d_k == nullptr || c->d_v == nullptr) return set_error(JQ_ERR_INVALID_ARG, "kv cache: null pointer");
    if (c->num_seqs > 0 && c->max_pages > 0 && c->d_page_table == nullptr) return set_error(JQ_ERR_INVALID_ARG, "kv cache: null page table");
    if (c->table_stride < c->max_pages && c->num_seqs > 1)
        return set_error(JQ_ERR_INVALID_ARG, "kv cache: rows of the page table overlap");
    const int64_t size = kv_element_bytes(c->type);
    const int64_t strides[3] = {c->stride_page, c->stride_slot, c->stride_head};
    const int64_t counts[3] = {c->num_pages, c->page_size, c->num_kv_heads};
    for (int i = 0; i < 3; ++i) {
        if (counts[i] == 1) continue;
        if (strides[i] < c->head_dim) return set_error(JQ_ERR_INVALID_ARG, "kv cache: rows overlap (a stride of %lld)", (long long)strides[i]);
        if (strides[i] > ((int64_t)1 << 60) / counts[i]) return set_error(JQ_ERR_TOO_LARGE, "kv cache: strides beyond 2^60 elements");
        if (strides[i] * size % 16 != 0) return set_error(JQ_ERR_ALIGN, "kv cache: strides must be multiples of 16 bytes");
    }
    if ((((uintptr_t)c->d_k | (uintptr_t)c->d_v) & 15u) != 0) return set_error(JQ_ERR_ALIGN, "kv cache: keys and values must be 16-byte aligned");
    if (((uintptr_t)c->d_page_table & 3u) != 0) return set_error(JQ_ERR_ALIGN, "kv cache: the page table must be 4-byte aligned");
    if (!(c->k_scale > 0.f) || !(c->v_scale > 0.f) || !std::isfinite(c->k_scale) || !std::isfinite(c->v_scale))
        return set_error(JQ_ERR_INVALID_ARG, "kv cache: scales must be positive and finite");
    ix->table = c->d_page_table;
    ix->table_stride = c->table_stride;
    ix->stride_page = c->num_pages == 1 ? 0 : c->stride_page;
    ix->stride_slot = c->page_size == 1 ? 0 : c->stride_slot;
    ix->stride_head = c->num_kv_heads == 1 ? 0 : c->stride_head;
    ix->num_seqs = (int32_t)c->num_seqs;
    ix->max_pages = (int32_t)c->max_pages;
    ix->num_pages = (int32_t)c->num_pages;
    kv_set_page_size(*ix, (int32_t)c->page_size);
    return JQ_OK;
}

}  // namespace jq

using namespace jq;

extern "C" {

int jq_rope_table_from(const double *radians, int64_t n_pairs, uint64_t *table_out) {
    if (n_pairs < 0 || (n_pairs > 0 && (radians == nullptr || table_out == nullptr)))
        return set_error(JQ_ERR_INVALID_ARG, "rope table: null pointer or negative size");
    for (int64_t i = 0; i < n_pairs; ++i) {
        if (!std::isfinite(radians[i])) return set_error(JQ_ERR_INVALID_ARG, "rope table: frequency %lld is not finite", (long long)i);
    }
    for (int64_t i = 0; i < n_pairs; ++i) table_out[i] = steps_of((long double)radians[i]);
    return JQ_OK;
}

int jq_rope_table(int64_t rotary_dim, double base, int scaling, double factor, int64_t original_length, uint64_t *table_out,
                  float *mscale_out) {
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > 1024)
        return set_error(JQ_ERR_SHAPE, "rope table: rotary_dim = %lld is not an even number up to 1024", (long long)rotary_dim);
    if (table_out == nullptr || mscale_out == nullptr) return set_error(JQ_ERR_INVALID_ARG, "rope table: null pointer");
    if (!(base > 1.0) || !std::isfinite(base)) return set_error(JQ_ERR_INVALID_ARG, "rope table: base must be above 1");
    if (scaling < JQ_ROPE_NONE || scaling > JQ_ROPE_WAVELENGTH) return set_error(JQ_ERR_INVALID_ARG, "rope table: unknown scaling %d", scaling);
    if (scaling != JQ_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
        return set_error(JQ_ERR_INVALID_ARG, "rope table: factor must be 1 or more");
    if ((scaling == JQ_ROPE_YARN || scaling == JQ_ROPE_WAVELENGTH) && original_length <= 0)
        return set_error(JQ_ERR_INVALID_ARG, "rope table: original_length must be positive");
    constexpr long double TWO_PI = 6.283185307179586476925286766559L;
    const long double r = (long double)rotary_dim;
    long double b = base;
    if (scaling == JQ_ROPE_NTK) b *= powl(factor, r / (r > 2 ? r - 2 : 1));
    if (!(b <= 1.7976931348623157e308L)) return set_error(JQ_ERR_INVALID_ARG, "rope table: the scaled base is not finite");
    long double low = 0, high = 0;
    if (scaling == JQ_ROPE_YARN) {
        // the pair that turns so many times within the original length
        const auto pair_of = [&](long double turns) { return r * logl((long double)original_length / (turns * TWO_PI)) / (2 * logl(b)); };
        low = fmaxl(floorl(pair_of(32)), 0);
        high = fminl(ceill(pair_of(1)), r - 1);
    }
    for (int64_t i = 0; i < rotary_dim / 2; ++i) {
        const long double f = powl(b, -2 * (long double)i / r);
        long double divided = 0;  // the share of the pair that is divided by the factor
        if (scaling == JQ_ROPE_LINEAR) divided = 1;
        if (scaling == JQ_ROPE_YARN) divided = fminl(fmaxl(((long double)i - low) / fmaxl(high - low, 0.001L), 0), 1);
        if (scaling == JQ_ROPE_WAVELENGTH) divided = 1 - fminl(fmaxl(((long double)original_length * f / TWO_PI - 1) / 3, 0), 1);
        // (f by itself also where there is no factor)
        table_out[i] = steps_of(divided == 0 ? f : f / factor * divided + f * (1 - divided));
    }
    *mscale_out = scaling == JQ_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.f;
    return JQ_OK;
}

int jq_rope_device(void *stream, const float *d_x, float *d_out, const int32_t *d_positions, const uint64_t *d_table,
                   int64_t num_rows, int64_t num_heads, int64_t head_dim, int64_t rotary_dim, int64_t x_stride_row,
                   int64_t x_stride_head, int64_t out_stride_row, int64_t out_stride_head, int interleaved, float mscale) {
    if (int rc = check_rope(num_rows, num_heads, head_dim, rotary_dim, mscale)) return rc;
    if (num_rows == 0 || num_heads == 0) return JQ_OK;
    if (d_x == nullptr || d_out == nullptr || d_positions == nullptr || d_table == nullptr)
        return set_error(JQ_ERR_INVALID_ARG, "rope: null pointer");
    if ((((uintptr_t)d_x | (uintptr_t)d_out | (uintptr_t)d_positions) & 3u) != 0 || ((uintptr_t)d_table & 7u) != 0)
        return set_error(JQ_ERR_ALIGN, "rope: heads and positions must be 4-byte, the table 8-byte aligned");
    if ((num_rows > 1 && out_stride_row < head_dim) || (num_heads > 1 && out_stride_head < head_dim))
        return set_error(JQ_ERR_INVALID_ARG, "rope: heads of the output overlap");
    RopeArgs a = {};
    a.x = d_x, a.x_row = x_stride_row, a.x_head = x_stride_head;
    a.out = d_out, a.out_row = out_stride_row, a.out_head = out_stride_head;
    a.positions = d_positions, a.table = reinterpret_cast<const unsigned long long *>(d_table);
    a.rows = (int)num_rows, a.heads = (int)num_heads, a.dim = (int)head_dim, a.half = (int)(rotary_dim / 2), a.mscale = mscale;
    return launch_rope<void>(static_cast<cudaStream_t>(stream), a, (int)rotary_dim, interleaved);
}

int jq_rope_kv_append_device(void *stream, const float *d_qkv, int64_t qkv_stride, float *d_q, int64_t q_stride_row,
                             int64_t q_stride_head, const int32_t *d_positions, const int32_t *d_index, const int32_t *d_seqs,
                             const uint64_t *d_table, int64_t rotary_dim, int64_t num_rows, int64_t num_q_heads,
                             const jq_kv_cache *cache, int interleaved, float mscale) {
    RopeArgs a = {};
    if (int rc = check_kv_cache(cache, &a.ix)) return rc;
    if (int rc = check_rope(num_rows, num_q_heads, cache->head_dim, rotary_dim, mscale)) return rc;
    const int64_t dim = cache->head_dim, all_heads = num_q_heads + 2 * cache->num_kv_heads;
    if (num_rows == 0) return JQ_OK;
    if (d_qkv == nullptr || d_positions == nullptr || d_index == nullptr || d_table == nullptr || (num_q_heads > 0 && d_q == nullptr))
        return set_error(JQ_ERR_INVALID_ARG, "rope append: null pointer");
    if ((((uintptr_t)d_qkv | (uintptr_t)d_q | (uintptr_t)d_positions | (uintptr_t)d_index | (uintptr_t)d_seqs) & 3u) != 0 ||
        ((uintptr_t)d_table & 7u) != 0)
        return set_error(JQ_ERR_ALIGN, "rope append: rows and indices must be 4-byte, the table 8-byte aligned");
    if (num_rows > 1 && qkv_stride < all_heads * dim) return set_error(JQ_ERR_INVALID_ARG, "rope append: rows of d_qkv overlap");
    if ((num_rows > 1 && num_q_heads > 0 && q_stride_row < dim) || (num_q_heads > 1 && q_stride_head < dim))
        return set_error(JQ_ERR_INVALID_ARG, "rope append: heads of d_q overlap");
    a.x = d_qkv, a.x_row = qkv_stride, a.x_head = dim;
    a.out = d_q, a.out_row = q_stride_row, a.out_head = q_stride_head;
    a.positions = d_positions, a.table = reinterpret_cast<const unsigned long long *>(d_table);
    a.rows = (int)num_rows, a.heads = (int)num_q_heads, a.kv_heads = (int)cache->num_kv_heads;
    a.dim = (int)dim, a.half = (int)(rotary_dim / 2), a.mscale = mscale;
    a.k = cache->d_k, a.v = cache->d_v, a.index = d_index, a.seqs = d_seqs;
    a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    a.fault = device_fault_ptr();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (cache->type) {
        case JQ_KV_F16: return launch_rope<KvF16>(st, a, (int)rotary_dim, interleaved);
        case JQ_KV_BF16: return launch_rope<KvBf16>(st, a, (int)rotary_dim, interleaved);
        default: return launch_rope<KvE4m3>(st, a, (int)rotary_dim, interleaved);
    }
}

}  // extern "C"
