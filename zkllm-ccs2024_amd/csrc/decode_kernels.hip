// Answering token by token in the prover's integers, for gfx950: the cache of keys and values, attention that reads it, and the logits' way to a token.
//
//   append     keys and values of new tokens to their places in the pages of their sequences
//   attention  x_j = q . k_j;  shift = the nearest integer to scale ln(sum_j exp(x_j / scale));  y_j = prod_i table_i[digit_i(shift - x_j)];
//              out = Q(Q(sum_j y_j v_j; s1); s2): the softmax of the layer's proof (zksoftmax.cu:4-32, :95-109, :112-173; self-attn.cu:81-98), the sum taken in
//              double precision and in the order of the keys as zk_softmax_shift takes it, so that results equal the class layer's
//   logits     penalties for repeated tokens, biases, the mask of a grammar, the best token that is left
//
// Positions, pages, lengths and tokens outside their ranges raise bits of a flag on the device; nothing is read or written out of range for them.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "detmath.hpp"
#include "intvalues.hpp"

using namespace zk;

// ---- the softmax --------------------------------------------------------------------------------------------------------------------------
static constexpr int DIGITS = 8;
struct SoftmaxArgs {
    const int32_t* table[DIGITS];        // of the digits that are kept, lowest first; null: 1 for digit 0 and 0 for others
    uint32_t radix[DIGITS];
    int bits[DIGITS];                    // log2 of the radices where all are powers of two
    int n, drop_bits;
    uint64_t drop;                       // the product of the radices whose digits are not kept
    double scale, scale_inv, scale_64;   // scale_64: 64 / (scale ln 2)
    // Two tables whose values need no gathers (a layer's): the first's by five terms of its series in the digit, to within `guard`, the second's from its first `live` entries, the others
    // being 0.  Digits of a distance d: bits from drop_bits on; d's upper half stays below upper_end.
    double series[5], guard;
    uint32_t live, upper_end;
};
struct SoftmaxPlan { SoftmaxArgs a; int32_t* memory = nullptr; bool pow2 = true, series = false; uint32_t dim = 0; };
static constexpr uint32_t MOST_LIVE = 8192;

__global__ void __launch_bounds__(256) k_softmax_table_i32(int32_t* __restrict__ table, double log_theta, double step, uint32_t len) {
    const uint32_t x = blockIdx.x * 256 + threadIdx.x;
    if (x < len) table[x] = (int32_t)(uint64_t)(zkd::exp_det(log_theta - step * (double)x) + 0.5);      // zk_softmax_table's values
}
// the weight of a key whose score lies d below the shift, below 2^47
template <bool POW2> __device__ __forceinline__ int64_t softmax_weight(int64_t d, const SoftmaxArgs& s, uint32_t& bad) {
    if (d < 0) { bad |= ZK_VALUES_TABLE; return 0; }
    uint64_t t = (uint64_t)d;
    int64_t y = 1;
    if constexpr (POW2) {
        t >>= s.drop_bits;
        for (int i = 0; i < s.n; ++i) {
            const uint32_t digit = (uint32_t)t & (s.radix[i] - 1);
            t >>= s.bits[i];
            y *= s.table[i] ? s.table[i][digit] : digit == 0 ? 1 : 0;
        }
    } else {
        t /= s.drop;
        for (int i = 0; i < s.n; ++i) {
            const uint32_t digit = (uint32_t)(t % s.radix[i]);
            t /= s.radix[i];
            y *= s.table[i] ? s.table[i][digit] : digit == 0 ? 1 : 0;
        }
    }
    if (t != 0) { bad |= ZK_VALUES_TABLE; return 0; }
    return y;
}

// ---- sequences and their pages ------------------------------------------------------------------------------------------------------------
struct Sequences {
    const int32_t *starts, *lengths;     // starts null: the same number of tokens each
    uint32_t count, tokens, max_length;
};
struct Sequence { uint32_t index, first, n, length; };
__device__ __forceinline__ bool sequence_at(const Sequences& s, uint32_t i, Sequence& q, uint32_t& bad) {
    q.index = i;
    if (s.starts) {
        const int32_t first = s.starts[i], end = s.starts[i + 1];
        if (first < 0 || end < first || (uint32_t)end > s.tokens) { bad |= ZK_VALUES_POSITION; return false; }
        q.first = (uint32_t)first; q.n = (uint32_t)(end - first);
    } else { q.n = s.tokens / s.count; q.first = i * q.n; }
    const int32_t length = s.lengths[i];
    if (length < 0 || (uint32_t)length > s.max_length) { bad |= ZK_VALUES_POSITION; return false; }
    q.length = (uint32_t)length;
    return true;
}
// the sequence that a token belongs to; none: tokens before the first and behind the last
__device__ __forceinline__ bool sequence_of(const Sequences& s, uint32_t token, Sequence& q, uint32_t& bad) {
    uint32_t i = 0;
    if (s.starts) {
        uint32_t lo = 0, hi = s.count;   // starts[lo] <= token or lo = 0
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (s.starts[mid] <= (int32_t)token) lo = mid;
            else hi = mid;
        }
        i = lo;
    } else i = token / (s.tokens / s.count);
    return sequence_at(s, i, q, bad) && token >= q.first && token - q.first < q.n;
}
// Where a token's heads lie in a cache, in two steps, so that the page is on its way while something else is done: its entry (without a table anything that can be read), then the place
struct Page { int32_t entry; uint32_t place; };
__device__ __forceinline__ Page page_of(const zk_i32_cache& c, uint32_t sequence, uint32_t t) {
    const uint32_t in = c.page_table ? t / c.page_size : 0;
    const int32_t* entry = c.page_table ? (const int32_t*)c.page_table + (size_t)sequence * c.table_cols + in : (const int32_t*)c.k;
    return Page{*entry, t - in * c.page_size};
}
__device__ __forceinline__ size_t cache_at(const zk_i32_cache& c, uint32_t sequence, const Page& p, uint32_t& bad) {
    const uint32_t page = c.page_table ? (uint32_t)p.entry : sequence;
    const bool has = page < c.pages;
    bad |= has ? 0u : (uint32_t)ZK_VALUES_POSITION;
    return (has ? page : 0u) * c.page_stride + p.place * c.token_stride;
}

// ---- append -------------------------------------------------------------------------------------------------------------------------------
struct AppendArgs {
    zk_i32_cache cache;
    const int32_t *k, *v;
    size_t k_token, k_head, v_token, v_head;
    uint32_t heads, dim;
    Sequences seqs;
    uint32_t* flag;
};
// A workgroup a token; HBM bounds many of them: 3200 tokens of 5 x 80, keys and values, 8.4 us, 2.4 TB/s, of which the launch is 2.3 (a single token's)
template <int VEC> __global__ void __launch_bounds__(256) k_cache_append(const AppendArgs a) {
    const uint32_t token = blockIdx.x, units = a.dim / VEC;
    uint32_t bad = 0;
    Sequence s;
    if (sequence_of(a.seqs, token, s, bad)) {
        const int64_t t = (int64_t)s.length - s.n + (token - s.first);
        if (t < 0) bad |= ZK_VALUES_POSITION;
        else {
            uint32_t off = 0;
            const size_t to = cache_at(a.cache, s.index, page_of(a.cache, s.index, (uint32_t)t), off);
            bad |= off;
            for (uint32_t i = threadIdx.x; !off && i < 2 * a.heads * units; i += 256) {
                const bool value = i >= a.heads * units;
                const uint32_t j = value ? i - a.heads * units : i, head = j / units, e = (j - head * units) * VEC;
                const int32_t* from = (value ? a.v + token * a.v_token + head * a.v_head : a.k + token * a.k_token + head * a.k_head) + e;
                int32_t* at = (int32_t*)(value ? a.cache.v : a.cache.k) + to + head * a.cache.head_stride + e;
                if constexpr (VEC == 4) *reinterpret_cast<v4i*>(at) = *reinterpret_cast<const v4i*>(from);
                else *at = *from;
            }
        }
    }
    if (threadIdx.x == 0) raise(a.flag, bad);
}

// ---- attention ----------------------------------------------------------------------------------------------------------------------------
// A row is one query head of a token; the rows of a head of keys are token * group + head in its group.  Four steps, each a launch: scores, a row's softmax to weights, sums of weights times
// values, and where the keys were cut into parts their sums joined.  Tiles are 16 or 64 rows: of the prefix's, any; of a sequence's own keys, its own.
// Scores are sums of 3 x 3 digit products (4 x 4 where a fourth digit is there), outputs of 5 x 3 (6 x 4), a digit product 2 * 16 * 16 * 64 operations in 16 cycles.  A prompt of 2048 tokens over as many keys,
// heads of 128, eight of them (of 32, 1.18 ms): splits 12 us, scores 69, the softmax 118 and 25 (the rows whose sums are taken in order), outputs 72.
// Keys and values of a part that many rows read, split into digits once for all of them: as the fragments of the matrix instructions, [head of keys][16 keys][64 dimensions][digit][lane][16] of the
// keys, [head of keys][64 keys][16 dimensions][digit][lane][16] of the values, and whether any of the 16 or 64 keys has a fourth digit
struct SplitPart { int8_t *k, *v; uint32_t *k_wide, *v_wide; };
struct AttnArgs {
    int32_t* out;
    const int32_t* q;
    size_t out_token, out_head, q_token, q_head;
    uint32_t group, dim, kv_heads, kv0;  // kv0: the launch's first head of keys
    SoftmaxArgs softmax;
    zk_i32_cache prefix, own;
    uint32_t prefix_len, prefix_cols;    // prefix_cols: the prefix's length up to a multiple of 64, where a row's own keys begin
    Sequences seqs;                      // count 0: no own keys
    int causal;
    Divisor sf_first, sf_second;
    int64_t* scores;                     // [head of keys][row][ld]
    int8_t* weights;                     // [head of keys][row][six digits][ld]
    uint32_t* top;                       // [head of keys][row]: the sixth digit is not all zeros
    uint32_t* unsure;                    // how many rows need their sum in order, three words, the rows
    size_t ld;                           // a multiple of 64
    int64_t* shift_out;                  // [token][head], or null
    int64_t* parts;                      // [split][head of keys][row][dim]: sums' sizes
    uint32_t* parts_low;                 // as many: their low 32 bits
    int direct;                          // the keys are one part: its sums are the outputs
    SplitPart split[2];                  // of the prefix and of the own keys
    uint32_t split_tiles[2];             // of 16 keys, a multiple of four
    uint32_t tokens, heads_here, prefix_tiles, prefix_splits, prefix_step, own_splits, own_step, score_keys;
    uint32_t* flag;
};
__device__ __forceinline__ uint32_t own_seen(const AttnArgs& a, const Sequence& s, uint32_t token) {      // how many of its sequence's own keys a token sees
    if (!a.causal) return s.length;
    const int64_t seen = (int64_t)s.length - s.n + (token - s.first) + 1;
    return seen < 0 ? 0u : (uint32_t)seen;
}
static constexpr uint32_t MOST_STEP = 8192;      // keys of a part: four products of 2^14 each in an accumulator of 32 bits
struct Tile {
    uint32_t row0, lo, hi, keys, col0;   // rows lo .. hi - 1 of those from row0 on are its own; keys: the most that one of them sees, behind column col0
    bool own;
    Sequence s;
    __device__ bool has(uint32_t c) const { return row0 + c >= lo && row0 + c < hi; }
};
// tile `id` of ROWS rows, of the prefix or of the sequences' own keys
template <uint32_t ROWS> __device__ __forceinline__ bool tile_at(const AttnArgs& a, bool own, uint32_t id, Tile& t, uint32_t& bad) {
    t.own = own;
    if (!own) {
        t.row0 = id * ROWS; t.lo = 0; t.hi = a.tokens * a.group; t.keys = a.prefix_len; t.col0 = 0;
        if (a.seqs.starts) {             // tokens before the first sequence and behind the last are nobody's
            const int32_t first = a.seqs.starts[0], end = a.seqs.starts[a.seqs.count];
            t.lo = (uint32_t)max(first, 0) * a.group; t.hi = min((uint32_t)max(end, 0), a.tokens) * a.group;
        }
        t.lo = max(t.lo, t.row0); t.hi = min(t.hi, t.row0 + ROWS);
        return t.lo < t.hi;
    }
    // A sequence's tiles begin at floor(first row / ROWS) + its index: a place for each of them, since floor(x + y) + 1 >= floor(x) + ceil(y)
    auto base = [&](uint32_t i) { return (uint32_t)((uint64_t)(a.seqs.starts ? (uint32_t)a.seqs.starts[i] : i * (a.tokens / a.seqs.count)) * a.group / ROWS) + i; };
    uint32_t lo = 0, hi = a.seqs.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (base(mid) <= id) lo = mid;
        else hi = mid;
    }
    if (!sequence_at(a.seqs, lo, t.s, bad)) return false;
    const uint32_t b = base(lo), rows = t.s.n * a.group, at = (id - b) * ROWS;
    if (id < b || at >= rows) return false;
    t.row0 = t.lo = t.s.first * a.group + at; t.hi = t.lo + min(ROWS, rows - at); t.col0 = a.prefix_cols;
    t.keys = own_seen(a, t.s, (t.hi - 1) / a.group);
    return true;
}
// How heads are read: an element at a time, four at a time, or four at a time with all 64 dimensions of every block there
enum class Heads { ANY, FOURS, BLOCKS };
// 16 of a head's values for its digit planes: four runs of four, 16 apart, so that four lanes read 64 bytes in one piece.  Which 16 of 64 a lane has is the same for queries and keys.  Beyond
// the head's end queries are zeros (ZEROS), keys anything.
template <Heads HEADS, bool ZEROS> __device__ __forceinline__ void head_piece(const int32_t* p, uint32_t d0, uint32_t dim, int32_t (&x)[16]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t d = d0 + 16 * w;
        if constexpr (HEADS == Heads::ANY) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int32_t v = p[min(d + e, dim - 1)];
                x[4 * w + e] = ZEROS && d + e >= dim ? 0 : v;
            }
        } else {
            const v4i v = *reinterpret_cast<const v4i*>(p + (HEADS == Heads::BLOCKS ? d : min(d, dim - 4)));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * w + e] = ZEROS && HEADS == Heads::FOURS && d >= dim ? 0 : v[e];
        }
    }
}
// four neighbouring dimensions from d on, beyond the head's end anything
template <Heads HEADS> __device__ __forceinline__ v4i four_of(const int32_t* p, uint32_t d, uint32_t dim) {
    if constexpr (HEADS == Heads::ANY) return v4i{p[min(d, dim - 1)], p[min(d + 1, dim - 1)], p[min(d + 2, dim - 1)], p[min(d + 3, dim - 1)]};
    else return *reinterpret_cast<const v4i*>(p + (HEADS == Heads::BLOCKS ? d : min(d, dim - 4)));
}
__device__ __forceinline__ bool any_bits(const v4i& v) { return (v[0] | v[1] | v[2] | v[3]) != 0; }

// A key's place among the 16 of a fragment, and the other way round: row 4 q + e of a product is key 2 q + e, or 8 + 2 q + e - 2, so that four lanes store 64 bytes of scores in one piece
__device__ __forceinline__ uint32_t key_of_lane(uint32_t c) { return (c >> 2) * 2 + (c & 1u) + (c & 2u) * 4; }
// A workgroup splits 64 keys of a head: a wave 16 keys, and the values of 64 dimensions.  HBM: 2048 keys of 8 heads of 128 in 11.5 us, 3.3 TB/s read and written
template <Heads HEADS> __global__ void __launch_bounds__(256) k_attn_split(const AttnArgs a, int own) {
    uint32_t bad = 0;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4, kv = a.kv0 + blockIdx.x, blocks = (a.dim + 63) / 64, units = blocks == 3 ? 4 : blocks, key0 = blockIdx.y * 64;
    uint32_t keys = a.prefix_len;
    Sequence s;
    if (own) {
        if (!sequence_at(a.seqs, 0, s, bad)) { raise(a.flag, bad); return; }
        keys = s.length;
    }
    if (key0 >= keys) return;
    const zk_i32_cache& cache = own ? a.own : a.prefix;
    const SplitPart& part = a.split[own];
    const uint32_t tiles = a.split_tiles[own];
    const Page k_page = page_of(cache, 0, min(key0 + wave * 16 + key_of_lane(c), keys - 1)), v_page = page_of(cache, 0, min(key0 + lane, keys - 1));
    {
        const int32_t* p = (const int32_t*)cache.k + kv * cache.head_stride + cache_at(cache, 0, k_page, bad);
        const size_t tile = (size_t)blockIdx.x * tiles + blockIdx.y * 4 + wave;
        bool wide = false;
        for (uint32_t u = 0; u < units; ++u) {             // as many blocks of dimensions as the scores' kernels take
            int32_t x[16];
            head_piece<HEADS, false>(p, u * 64 + q * 4, a.dim, x);
            v4i d[4];
            digit_planes(x, d, bad);
            wide |= any_bits(d[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<v4i*>(part.k + ((tile * units + u) * 4 + j) * 1024 + lane * 16) = d[j];
        }
        const bool any = __any(wide);
        if (lane == 0) part.k_wide[tile] = any;
    }
    __shared__ uint32_t v_wide;
    if (threadIdx.x == 0) v_wide = 0;
    __syncthreads();
    for (uint32_t b = wave; b < blocks; b += 4) {
        const int32_t* values = (const int32_t*)cache.v + kv * cache.head_stride;
        const size_t mine = cache_at(cache, 0, v_page, bad);
        int32_t x[4][16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const v4i v = four_of<HEADS>(values + __shfl((unsigned long long)mine, (int)(q * 16 + i), 64), b * 64 + 4 * c, a.dim);
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n][i] = v[n];
        }
        const size_t at = (((size_t)blockIdx.x * (tiles / 4) + blockIdx.y) * blocks + b) * 4;
        bool wide = false;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            v4i d[4];
            digit_planes(x[n], d, bad);
            wide |= any_bits(d[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<v4i*>(part.v + ((at + n) * 4 + j) * 1024 + lane * 16) = d[j];
        }
        if (__any(wide) && lane == 0) v_wide = 1;
    }
    __syncthreads();
    if (threadIdx.x == 0) part.v_wide[(size_t)blockIdx.x * (tiles / 4) + blockIdx.y] = v_wide;
    raise(a.flag, bad);
}
// Scores: a wave takes 16 keys by 16 RT rows at a time, a lane 16 of 64 dimensions of one of the keys, straight from memory to the fragments of v_mfma_i32_16x16x64_i8.  The next keys are
// on their way while these are multiplied, and the place of those behind them is looked up.  Few rows wait for memory: 16000 keys of 8 heads of 128, 4 rows each, 17 us, 3.9 TB/s.  Many rows are bound by
// issue, splitting keys as much as joining sums: 128 rows over 8192 keys 41 us, 0.94 POP/s (two workgroups a
// unit, with registers spilled: 46); with keys split before (SPLIT), 2048 over 2048, 69 us, 1.1 POP/s.  Half as many rows a wave (RT 2) gain nothing.
template <int U, int RT, Heads HEADS, int WAVES, bool SPLIT> __device__ __forceinline__ void scores_of(const AttnArgs& a, const Tile& t, uint32_t kv, uint32_t first, uint32_t end, v4i (&fourth)[RT][U][64],
                                                                                                 int64_t* out, size_t ld, uint32_t& bad) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4;
    auto query = [&](int r, int u, v4i (&d)[4]) {
        const uint32_t row = t.has(16 * r + c) ? t.row0 + 16 * r + c : t.lo, token = row / a.group, head = kv * a.group + (row - token * a.group);
        int32_t x[16];
        head_piece<HEADS, true>(a.q + token * a.q_token + head * a.q_head, u * 64 + q * 4, a.dim, x);
        digit_planes(x, d, bad);
    };
    const zk_i32_cache& cache = t.own ? a.own : a.prefix;
    const int32_t* keys = (const int32_t*)cache.k + kv * cache.head_stride;
    const uint32_t my_key = key_of_lane(c), sequence = t.own ? t.s.index : 0u;
    auto page = [&](uint32_t key) { return page_of(cache, sequence, min(key + my_key, t.keys - 1)); };
    int32_t x[SPLIT ? 1 : U][16];
    v4i planes[SPLIT ? U : 1][3];
    uint32_t wide_next = 0;
    const size_t tile0 = SPLIT ? (size_t)(kv - a.kv0) * a.split_tiles[t.own] : 0;
    auto fetch = [&](const Page& at, uint32_t key) {
        if constexpr (SPLIT) {
            const size_t tile = tile0 + key / 16;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int m = 0; m < 3; ++m) planes[u][m] = *reinterpret_cast<const v4i*>(a.split[t.own].k + ((tile * U + u) * 4 + m) * 1024 + lane * 16);
            wide_next = a.split[t.own].k_wide[tile];
        } else {
            const int32_t* p = keys + cache_at(cache, sequence, at, bad);
#pragma unroll
            for (int u = 0; u < U; ++u) head_piece<HEADS, false>(p, u * 64 + q * 4, a.dim, x[u]);
        }
    };
    uint32_t key = first + wave * 16;
    Page next{0, 0};
    if constexpr (!SPLIT) next = page(key + WAVES * 16);
    if (key < end) fetch(SPLIT ? next : page(key), key);
    v4i b[RT][U][3];
    bool wide = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v4i d[4];
            query(r, u, d);
#pragma unroll
            for (int m = 0; m < 3; ++m) b[r][u][m] = d[m];
            fourth[r][u][lane] = d[3];                     // rarely needed; every wave has the same
            wide |= any_bits(d[3]);
            if ((r * U + u) % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // more of them at once crowd the registers
        }
    }
    const bool q_wide = __any(wide);
    int64_t* const to0 = out + c * ld + 2 * q;
    for (; key < end; key += WAVES * 16) {
        v4i k[U][SPLIT ? 3 : 4];
        bool k_wide = false;
        if constexpr (SPLIT) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int m = 0; m < 3; ++m) k[u][m] = planes[u][m];
            k_wide = wide_next != 0;
            if (key + WAVES * 16 < end) fetch(next, key + WAVES * 16);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                digit_planes(x[u], k[u], bad);
                k_wide |= any_bits(k[u][3]);
            }
            const Page after = page(key + 2 * WAVES * 16);
            if (key + WAVES * 16 < end) fetch(next, 0);
            next = after;
        }
        const bool four = q_wide || __any(k_wide);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            v4i acc[5];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 9; ++i) {              // in an order that adds to no sum twice in a row
                    constexpr int M[9] = {0, 0, 0, 1, 2, 1, 1, 2, 2}, N[9] = {0, 1, 2, 2, 2, 0, 1, 1, 0};
                    const int sum = M[i] + N[i];
                    acc[sum] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[u][M[i]], b[r][u][N[i]], u == 0 && i < 5 ? v4i{0, 0, 0, 0} : acc[sum], 0, 0, 0);
                }
            int64_t v[4];
            if (!four) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (U <= 2) v[e] = (int64_t)(acc[2][e] + acc[3][e] * 256) * 65536 + ((int64_t)(acc[0][e] + acc[1][e] * 256) + ((int64_t)acc[4][e] << 32));      // two products of 2^14 in 128 dimensions
                    else v[e] = acc[0][e] + (int64_t)acc[1][e] * 256 + (acc[2][e] + (int64_t)acc[3][e] * 256) * 65536 + ((int64_t)acc[4][e] << 32);
                }
            } else {
                v4i more[3] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};      // of 256^4 on, but for 256^3
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const v4i d3 = fourth[r][u][lane];
                    v4i k3;
                    if constexpr (SPLIT) k3 = *reinterpret_cast<const v4i*>(a.split[t.own].k + (((tile0 + key / 16) * U + u) * 4 + 3) * 1024 + lane * 16);
                    else k3 = k[u][3];
#pragma unroll
                    for (int m = 0; m < 3; ++m) {
                        v4i& to = m == 0 ? acc[3] : m == 1 ? more[0] : more[1];
                        to = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[u][m], d3, to, 0, 0, 0);
                        to = __builtin_amdgcn_mfma_i32_16x16x64_i8(k3, b[r][u][m], to, 0, 0, 0);
                    }
                    more[2] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k3, d3, more[2], 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t s[7] = {acc[0][e], acc[1][e], acc[2][e], acc[3][e], acc[4][e] + more[0][e], more[1][e], more[2][e]};
                    v[e] = joined<7>(s, bad);
                }
            }
            if (!t.has(16 * r + c)) continue;
            typedef long long v2l __attribute__((ext_vector_type(2)));
            v2l* to = reinterpret_cast<v2l*>(to0 + 16 * r * ld + key);
            to[0] = v2l{v[0], v[1]};
            to[4] = v2l{v[2], v[3]};
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}
template <int U, int RT, Heads HEADS, bool SPLIT> __global__ void __launch_bounds__(256, RT > 1 ? 1 : 2) k_attn_scores(const AttnArgs a, int own) {
    __shared__ v4i fourth[RT][U][64];
    uint32_t bad = 0;
    Tile t;
    if ((blockIdx.y | blockIdx.z | blockIdx.x | threadIdx.x) == 0) *a.unsure = 0;
    if (!tile_at<16 * RT>(a, own, blockIdx.z, t, bad)) { raise(a.flag, bad); return; }
    const uint32_t key0 = blockIdx.y * a.score_keys;
    if (key0 >= t.keys) return;
    scores_of<U, RT, HEADS, 4, SPLIT>(a, t, a.kv0 + blockIdx.x, key0, min(key0 + a.score_keys, t.keys), fourth, a.scores + ((size_t)blockIdx.x * a.tokens * a.group + t.row0) * a.ld + t.col0, a.ld, bad);
    raise(a.flag, bad);
}

// The sum of a row's exponentials in double precision and in the order of the keys, by many lanes.  As long as the sum t stays below a power of two 2^(e + 1), adding a term x
// to it adds the whole number of units u = 2^(e - 52) that is nearest to x / u, and of two that are equally near the one that leaves t / u even: what a run of terms adds
// depends on nothing of t but whether t / u is odd.  Such pairs of sums, for even and for odd t / u, are joined in any grouping.  Where the sum would leave 2^(e + 1) -- some fifteen
// times in a row of thousands -- the lanes before the one where it does are added so and that lane's terms one by one.
struct Steps { uint64_t even, odd; };
__device__ __forceinline__ Steps then(const Steps& a, const Steps& b) { return Steps{a.even + (a.even & 1 ? b.odd : b.even), a.odd + (a.odd & 1 ? b.even : b.odd)}; }
static constexpr uint64_t UNITS = 0x0020000000000000ull;                       // t / u stays below
__device__ __forceinline__ int exponent(double t) { return (int)(zkd::double_to_bits(t) >> 52) - 1023; }
__device__ __forceinline__ uint64_t units_of(double t) { return (zkd::double_to_bits(t) & 0x000FFFFFFFFFFFFFull) | 0x0010000000000000ull; }
__device__ __forceinline__ void step(Steps& s, double x, int e) {
    const double w = __builtin_fmin(ldexp(x, 52 - e), 4503599627370496.0);     // 2^52 of them leave 2^(e + 1) already
    const double near = w + 4503599627370496.0;                                // rounds to whole numbers, ties to even ones
    const uint64_t units = zkd::double_to_bits(near) - 0x4330000000000000ull;
    const double rest = w - (near - 4503599627370496.0);
    const bool tie = rest == 0.5 || rest == -0.5;
    const uint64_t other = tie ? (rest > 0 ? 1ull : ~0ull) : 0ull;             // to the odd neighbour
    s.even += units + (s.even & 1 ? other : 0);
    s.odd += units + (s.odd & 1 ? 0 : other);
}
// steps over the lanes up to this one
__device__ __forceinline__ Steps steps_up_to(Steps s) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const Steps before{__shfl_up(s.even, off, 64), __shfl_up(s.odd, off, 64)};
        const Steps both = then(before, s);
        if (lane >= (uint32_t)off) s = both;
    }
    return s;
}
// steps over the lanes from this one on
__device__ __forceinline__ Steps steps_from(Steps s) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const Steps behind{__shfl_down(s.even, off, 64), __shfl_down(s.odd, off, 64)};
        const Steps both = then(s, behind);
        if (lane + (uint32_t)off < 64) s = both;
    }
    return s;
}
__device__ __forceinline__ uint64_t of_lane(uint64_t x, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), (int)lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, (int)lane);
}
__device__ __forceinline__ double of_lane(double x, uint32_t lane) { return zkd::bits_to_double(of_lane(zkd::double_to_bits(x), lane)); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
}
// total with the terms of 64 lanes added, lane by lane, M in a lane
template <int M> __device__ __forceinline__ double add_in_order(double total, const double (&x)[M]) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t from = 0;                         // lanes before this one are in the total
    while (true) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < M; ++i) any |= x[i] != 0.0;
        const unsigned long long left = __ballot(any && lane >= from);
        if (left == 0 || !(total < __builtin_inf())) return total;
        uint32_t at = (uint32_t)__builtin_ctzll(left), until = min(at + 64 / M, 64u);      // a row's first terms: every few of them leave a power of two
        if (total > 0.0) {
            const int e = exponent(total);
            const uint64_t t = units_of(total);
            Steps s{0, 0};
            if (lane >= from)
#pragma unroll
                for (int i = 0; i < M; ++i) step(s, x[i], e);
            s = steps_up_to(s);
            const uint64_t after = t + (t & 1 ? s.odd : s.even);
            const unsigned long long out = __ballot(after >= UNITS);
            const uint32_t last = out ? (uint32_t)__builtin_ctzll(out) : 64u;      // the lane where the sum leaves 2^(e + 1)
            if (last > 0) {
                const uint64_t sum = __shfl(after, last - 1, 64);
                total = ldexp((double)sum, e - 52);
            }
            if (last == 64) return total;
            at = last;
            until = at + 1;
        }
        for (; at < until; ++at)
#pragma unroll
            for (int i = 0; i < M; ++i) total = total + of_lane(x[i], at);
        from = until;
        if (from == 64) return total;
    }
}
// (double)x / scale, correctly rounded: two corrections of x / scale's estimate by the scale's correctly rounded inverse, the first of which leaves less than a unit in the last place,
// from where the second rounds correctly
__device__ __forceinline__ double divided(int64_t x, double scale, double scale_inv) {
    const double v = (double)x;
    double q = v * scale_inv;
    q = __builtin_fma(__builtin_fma(-q, scale, v), scale_inv, q);
    return __builtin_fma(__builtin_fma(-q, scale, v), scale_inv, q);
}
// weights as digits: of eight keys, a plane's eight bytes at a time
struct Digits8 { uint2 p[6]; };
__device__ __forceinline__ void digits8(const uint64_t (&d)[8], Digits8& out) {      // d: digits in bytes 0 .. 5
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { lo[e] = (uint32_t)d[4 * w + e]; hi[e] = (uint32_t)(d[4 * w + e] >> 32); }
        const uint32_t a = __builtin_amdgcn_perm(lo[1], lo[0], 0x05010400u), b = __builtin_amdgcn_perm(lo[1], lo[0], 0x07030602u);
        const uint32_t c = __builtin_amdgcn_perm(lo[3], lo[2], 0x05010400u), f = __builtin_amdgcn_perm(lo[3], lo[2], 0x07030602u);
        const uint32_t g = __builtin_amdgcn_perm(hi[1], hi[0], 0x05010400u), h = __builtin_amdgcn_perm(hi[3], hi[2], 0x05010400u);
        const uint32_t v[6] = {__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u), __builtin_amdgcn_perm(f, b, 0x05040100u),
                               __builtin_amdgcn_perm(f, b, 0x07060302u), __builtin_amdgcn_perm(h, g, 0x05040100u), __builtin_amdgcn_perm(h, g, 0x07060302u)};
#pragma unroll
        for (int j = 0; j < 6; ++j) (w ? out.p[j].y : out.p[j].x) = v[j];
    }
}
enum class Weights { ANY, POW2, SERIES };
enum class Sums { NEAR, IN_ORDER, BOTH };
static constexpr int64_t NO_KEY = INT64_MIN;      // a score whose exponential is 0: scales are 2^53 at most
// a b + c with c in scalar registers: the compiler copies a constant to vector registers for every addition otherwise
__device__ __forceinline__ double fma_s(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}
// exp(v / scale) to some 2^-50 and what v / scale's rounding adds: 2^(n / 64) out of LDS and five terms behind it
__device__ __forceinline__ double exp_near(int64_t v, const SoftmaxArgs& s, const double* power) {
    const double x = (double)v * s.scale_64, n = rint(x), f = x - n;
    constexpr double L = 0.69314718055994530942 / 64.0;
    double p = fma_s(f, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
    p = fma_s(f, p, L * L * L / 6.0);
    p = fma_s(f, p, L * L / 2.0);
    p = fma_s(f, p, L);
    p = __builtin_fma(f, p, 1.0);
    int i;                               // far beyond what a double's exponent holds the largest or smallest of its type
    asm("v_cvt_i32_f64 %0, %1" : "=v"(i) : "v"(n));
    return ldexp(power[i & 63] * p, i >> 6);
}
// zkd::exp_det(x) operation for operation, without branches and with the constants in scalar registers
__device__ __forceinline__ double exp_exact(double x) {
    const double at = __builtin_fmin(__builtin_fmax(x, -708.0), 709.0);
    const double kf = at * 1.44269504088896338700e+00;
    const int k = (int)(kf + (kf >= 0 ? 0.5 : -0.5));
    const double kd = (double)k, r = __builtin_fma(-kd, 1.90821492927058770002e-10, __builtin_fma(-kd, 6.93147180369123816490e-01, at));
    double p = fma_s(r, 1.0 / 87178291200.0, 1.0 / 6227020800.0);
    p = fma_s(p, r, 1.0 / 479001600.0);
    p = fma_s(p, r, 1.0 / 39916800.0);
    p = fma_s(p, r, 1.0 / 3628800.0);
    p = fma_s(p, r, 1.0 / 362880.0);
    p = fma_s(p, r, 1.0 / 40320.0);
    p = fma_s(p, r, 1.0 / 5040.0);
    p = fma_s(p, r, 1.0 / 720.0);
    p = fma_s(p, r, 1.0 / 120.0);
    p = fma_s(p, r, 1.0 / 24.0);
    p = fma_s(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const double y = ldexp(p, k);              // exact: a normal number
    return x > 709.0 ? __builtin_inf() : x < -708.0 ? 0.0 : y;
}
// the columns of a row's scores: the prefix's, then, from a multiple of 64 on, its own
struct Columns {
    uint32_t prefix_len, prefix_cols, own_end, end;
    __device__ uint32_t keys_at(uint32_t j) const { return j < prefix_cols ? (j < prefix_len ? min(8u, prefix_len - j) : 0u) : j < own_end ? min(8u, own_end - j) : 0u; }      // of eight from j on
};
// n of eight scores, and in place of the others no keys
__device__ __forceinline__ void eight_scores(const int64_t* x, uint32_t n, int64_t (&v)[8]) {
    typedef long long v2l __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = NO_KEY;
    if (n == 0) return;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const v2l p = *reinterpret_cast<const v2l*>(x + i);
        v[i] = p[0]; v[i + 1] = p[1];
    }
    if (n < 8)
#pragma unroll
        for (int i = 1; i < 8; ++i) v[i] = i < (int)n ? v[i] : NO_KEY;
}
static constexpr int NO_EXPONENT = 2000;
template <int W> struct RowShared { double sums[W], partial[W], in_order[2]; Steps steps[W]; int at_exponent[W]; uint32_t any_top; };
// the sum of a row's exponentials in the order of the keys, by one wave
__device__ __forceinline__ double sum_in_order(const int64_t* x, const Columns& columns, double scale, double scale_inv) {
    const uint32_t lane = threadIdx.x & 63u;
    double t = 0.0;
    for (uint32_t j0 = 0; j0 < columns.end; j0 += 128) {      // few at a time: the registers hold a row's scores
        const uint32_t j = j0 + lane * 2, in8 = j & 7u, keys8 = columns.keys_at(j - in8), keys = keys8 > in8 ? keys8 - in8 : 0u;
        double term[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) term[e] = e < (int)keys ? zkd::exp_det(divided(x[j + e], scale, scale_inv)) : 0.0;
        t = add_in_order<2>(t, term);
    }
    return t;
}
// ... by W waves, 512 keys each at a time.  What a wave's terms do to the sum is made ready by all waves at once, for the power of two that the sum will be in, or the two, as sums in no order say; then the
// sum goes from wave to wave: over one that stays within its power of two in every wave at once, through one that leaves it up to the lane that does, that lane's terms and the lanes behind it, and through
// one that leaves several, as a row's first, by one
// power of two after the other (term by term each takes 35 cycles).
template <int W> __device__ __forceinline__ double sum_in_order(const int64_t* x, const Columns& columns, double scale, double scale_inv, RowShared<W>& sh) {
    constexpr int M = 8, T = 64 * W;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t slot = 0;
    double t = 0.0;
    for (uint32_t j0 = 0; j0 < columns.end; j0 += T * M) {
        const uint32_t j = j0 + threadIdx.x * M, keys = columns.keys_at(j);
        double term[M], mine = 0.0;
        int64_t v[M];
        eight_scores(x + j, keys, v);
#pragma unroll
        for (int e = 0; e < M; ++e) {
            term[e] = exp_exact(divided(v[e], scale, scale_inv));
            mine += term[e];
            if (e % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) mine += __shfl_xor(mine, off, 64);
        __syncthreads();
        if (lane == 0) sh.sums[wave] = mine;
        __syncthreads();
        double before = lane < wave ? sh.sums[lane] : 0.0;
#pragma unroll
        for (int off = 1; off < W; off <<= 1) before += __shfl_xor(before, off, 64);      // in the first W lanes
        before = t + of_lane(before, 0);
        const double behind = before + mine;
        // the powers of two that the sum can be in, by a margin that the sums' order cannot reach
        const bool known = before > 0.0 && behind < __builtin_inf();
        const int low = known ? exponent(before * (1.0 - 1e-9)) : NO_EXPONENT, high = known ? exponent(behind * (1.0 + 1e-9)) : NO_EXPONENT;
        const bool clean = known && low == high, one = known && low + 1 == high;
        Steps up{0, 0}, rest{0, 0};
        if (clean || one) {
#pragma unroll
            for (int k = 0; k < M; ++k) step(up, term[k], low);
            up = steps_up_to(up);
        }
        if (one) {
#pragma unroll
            for (int k = 0; k < M; ++k) step(rest, term[k], high);
            rest = steps_from(rest);
        }
        if (lane == 63) {
            sh.steps[wave] = up;
            sh.at_exponent[wave] = clean ? low : NO_EXPONENT;
        }
        __syncthreads();
        const int es = sh.at_exponent[lane % W];
        const Steps steps = sh.steps[lane % W];
#pragma unroll 1                          // code that is run once waits for its instructions
        for (uint32_t k = 0; k < (uint32_t)W; ++k) {
            // steps within a power of two are what they add to t's bits
            const uint64_t bits = uniform(zkd::double_to_bits(t));
            if (bits != 0 && (int)(bits >> 52) - 1023 == __builtin_amdgcn_readlane(es, (int)k)) {
                const uint64_t after = bits + (bits & 1 ? of_lane(steps.odd, k) : of_lane(steps.even, k));
                if (after >> 52 == bits >> 52) { t = zkd::bits_to_double(after); continue; }
            }
            if (wave == k) {
                bool added = false;
                if (one && t > 0.0 && exponent(t) == low) {
                    const uint64_t u = units_of(t), after = u + (u & 1 ? up.odd : up.even);
                    const unsigned long long out = __ballot(after >= UNITS);
                    const uint32_t last = out ? (uint32_t)__builtin_ctzll(out) : 64u;      // the lane where the sum leaves 2^(low + 1)
                    double r = last ? ldexp((double)__shfl(after, (int)last - 1, 64), low - 52) : t;
                    if (last < 64)
#pragma unroll
                        for (int i = 0; i < M; ++i) r = r + of_lane(term[i], last);
                    added = last >= 63;
                    if (!added && exponent(r) == high) {
                        const uint64_t v = units_of(r), even = __shfl(rest.even, (int)last + 1, 64), odd = __shfl(rest.odd, (int)last + 1, 64), end = v + (v & 1 ? odd : even);
                        added = end < UNITS;
                        r = ldexp((double)end, high - 52);
                    }
                    if (added) t = r;
                }
                if (!added) t = add_in_order<M>(t, term);
                if (lane == 0) sh.in_order[slot] = t;
            }
            __syncthreads();
            t = sh.in_order[slot];
            slot ^= 1;                     // the next writer does not wait until every wave has read this one
        }
    }
    return t;
}
// W waves a row, eight neighbouring keys a lane at a time.  The sum of exponentials is taken in no order first, from exponentials that are near: off from the sum in
// order by at most 2^-53 of all of that one's partial sums (half of the keys times the whole, where terms are alike) and what the exponentials are off.  That decides the shift unless it lies that near to a border between two whole numbers (one row in 65 at 2048 keys and
// a scale of 2^32 sqrt(128)); then the sum in order is taken -- by a launch of its own for such rows, where there are many rows --, the waves' runs at once where the sum stays within a power of
// two, and the few others one after the other.
// Latency bounds it where rows are few: 32 rows of 16000 keys 44 us, of it 9 for the tables and the near sum, 30 for the sum in order (dependent additions, scans and barriers; sixteen waves a row, with half
// the registers each: 51), 5 for the weights.  Memory and issue where they are many: 16384 rows of 2048 keys 118 us, scores read twice and weights written 6.2 TB/s, 63 instructions a score 43 % of the
// slots (four waves a row: 144; all of a row's scores held in registers instead of read a second time: 118; five waves a SIMD instead of four: 138), and 25 for the one row in 65 whose sum is taken in order.
// A row's scores x to its weights, zeros up to `fill`; ld from digit to digit.  false: its sum must be taken in order (SUMS NEAR)
template <int W, Weights KIND, Sums SUMS> __device__ __forceinline__ bool softmax_row(const SoftmaxArgs& s, const int64_t* x, int8_t* weights, size_t ld, const Columns& columns, uint32_t fill,
                                                                                      const int32_t* live, const double* power, RowShared<W>& sh, int64_t& shift, bool& top, uint32_t& bad) {
    constexpr int M = 8, T = 64 * W;
    const uint32_t lane = threadIdx.x & 63u, wave = W == 1 ? 0 : threadIdx.x >> 6, tid = wave * 64 + lane;
    const uint32_t stretches = (columns.end + T * M - 1) / (T * M);
    int64_t v[M];
    uint32_t n = 0;
    auto load = [&](uint32_t stretch) {
        const uint32_t j = stretch * T * M + tid * M;
        n = columns.keys_at(j);
        eight_scores(x + j, n, v);
    };
    auto rounded = [](double sv) { return sv >= 0 ? (int64_t)(sv + 0.5) : (int64_t)(sv - 0.5); };
    shift = 0;
    bool sure = columns.end == 0, loaded = false;
    if constexpr (SUMS != Sums::IN_ORDER) {
        double total = 0.0, partial = 0.0;            // partial: of all the sums on the way, each of which is rounded once
        for (uint32_t i = 0; i < stretches; ++i) {
            load(i);
            const double before = total;
#pragma unroll
            for (int e = 0; e < M; ++e) {
                total += exp_near(v[e], s, power);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // more of them at once crowd the registers
            }
            partial += (total - before) * (double)(columns.end - min(columns.end, i * T * M + tid * M));
        }
        loaded = stretches == 1;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { total += __shfl_xor(total, off, 64); partial += __shfl_xor(partial, off, 64); }
        if constexpr (W > 1) {
            __syncthreads();                           // the arrays' last use is over
            if (lane == 0) { sh.sums[wave] = total; sh.partial[wave] = partial; }
            __syncthreads();
            total = partial = 0.0;
#pragma unroll
            for (int i = 0; i < W; ++i) { total += sh.sums[i]; partial += sh.partial[i]; }
        }
        if (columns.end) {
            // The sum in order is off by 2^-53 of each sum on its way, this one by as much of the whole for each of a lane's terms, of which there are a 64th of the columns and 22 at most.  Both sums'
            // exponentials of x together are off by 1.2e-15 (4e-16 of exp_det twice, the rest roundings) and, by the roundings of x / scale, 4.8e-16 |x|; weighted by what they have in the sum t,
            // |x| is |ln t| + 17.4 at most (17.4: the logarithm of 2^25 keys).  Both logarithms are off by 4e-16 of them and their products with the scale by 2^-53.
            const double ln = zkd::log_det(total), sv = s.scale * ln;
            const double off = s.scale * ((partial / total + (double)(columns.end / 64 + 24)) * 1.2e-16 + 1.6e-15 * fabs(ln) + 1e-14), from_border = fabs(sv - floor(sv) - 0.5);
            sure = total > 1e-280 && total < 1e280 && off < 0.25 && from_border > off;
            if (sure) shift = rounded(sv);
        }
        if constexpr (SUMS == Sums::NEAR)
            if (!sure) return false;
    }
    if constexpr (SUMS != Sums::NEAR)
        if (!sure) {
            double sum;
            if constexpr (W == 1) sum = sum_in_order(x, columns, s.scale, s.scale_inv);
            else sum = sum_in_order<W>(x, columns, s.scale, s.scale_inv, sh);
            shift = rounded(s.scale * zkd::log_det(sum));
            loaded = false;                            // the registers were needed
        }
    // Both tables' values and their product are exact in double precision, and so is the number whose low 48 bits are the digits with 128 added to each
    constexpr double BASE = 4503599627370496.0 + 141289400074368.0;
    auto by_series = [&](int64_t score) {
        const uint64_t below = (uint64_t)(shift - score);
        const uint32_t lo = (uint32_t)below, hi = (uint32_t)(below >> 32), digit = lo >> s.drop_bits & (s.radix[0] - 1), upper = __builtin_amdgcn_alignbit(hi, lo, s.drop_bits + s.bits[0]);
        const bool reached = hi < s.upper_end;         // neither negative nor too far
        bad |= reached ? 0u : (uint32_t)ZK_VALUES_TABLE;
        const double z = (double)digit;
        const double u = fma_s(z, __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, s.series[4], s.series[3]), s.series[2]), s.series[1]), s.series[0]);
        double first = floor(u);
        if (fabs(u - first - 0.5) > 0.5 - s.guard) first = (double)s.table[0][digit];      // nearer to a border than the terms left out
        const int32_t second = live[min(upper, s.live - 1)];
        return __builtin_fma(first, reached && upper < s.live ? (double)second : 0.0, BASE);
    };
    top = false;
    const uint32_t fills = (fill + T * M - 1) / (T * M);
    for (uint32_t i = 0; i < fills; ++i) {
        if (!loaded || i != 0) load(i);
        {
            const uint32_t j = i * T * M + tid * M;
            if (j >= fill) continue;
            uint64_t d[M];
            if (n < M)
#pragma unroll
                for (int e = 0; e < M; ++e) v[e] = e < (int)n ? v[e] : shift;
#pragma unroll
            for (int e = 0; e < M; ++e) {
                if constexpr (KIND == Weights::SERIES) d[e] = zkd::double_to_bits(by_series(v[e])) ^ 0x808080808080ull;
                else d[e] = ((uint64_t)softmax_weight<KIND == Weights::POW2>(shift - v[e], s, bad) + 0x808080808080ull) ^ 0x808080808080ull;
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
            if (n < M)
#pragma unroll
                for (int e = 0; e < M; ++e) d[e] = e < (int)n ? d[e] : 0;
            Digits8 p;
            digits8(d, p);
            top |= (p.p[5].x | p.p[5].y) != 0;
#pragma unroll
            for (int k = 0; k < 6; ++k) *reinterpret_cast<uint2*>(weights + k * ld + j) = p.p[k];
        }
    }
    return true;
}
// the tables of a workgroup of THREADS lanes
template <int THREADS, Weights KIND> __device__ __forceinline__ void softmax_tables(const SoftmaxArgs& s, int32_t* live, double* power) {
    if constexpr (KIND == Weights::SERIES) {
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < s.live; i += THREADS) live[i] = s.table[1][i];
    }
    if (threadIdx.x < 64) power[threadIdx.x] = zkd::exp_det((double)threadIdx.x * (0.69314718055994530942 / 64.0));
}
template <int W, Weights KIND, Sums SUMS> __global__ void __launch_bounds__(W > 4 ? 64 * W : 256, SUMS == Sums::NEAR ? 4 : 1) k_attn_softmax(const AttnArgs a) {
    constexpr int T = 64 * W, ROWS = W > 4 ? 1 : 4 / W;    // a workgroup's rows at a time
    static_assert(W == 1 || ROWS == 1, "waves that share a row meet at the workgroup's barriers");
    extern __shared__ int32_t live[];
    __shared__ double power[64];
    __shared__ RowShared<W> sh;
    const uint32_t rows = a.tokens * a.group, all = a.heads_here * rows, lane = threadIdx.x & 63u, tid = W == 1 ? lane : threadIdx.x;
    uint32_t bad = 0;
    softmax_tables<T * ROWS, KIND>(a.softmax, live, power);
    __syncthreads();
    const uint32_t work = SUMS == Sums::IN_ORDER ? *a.unsure : all;
    for (uint32_t at = W == 1 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * ROWS + (threadIdx.x >> 6))) : blockIdx.x; at < work; at += gridDim.x * ROWS) {
        const uint32_t r = SUMS == Sums::IN_ORDER ? a.unsure[4 + at] : at, in = r % rows, token = in / a.group;
        int8_t* weights = a.weights + (size_t)r * 6 * a.ld;
        uint32_t own = 0;
        Sequence q;
        if (a.seqs.count) {
            if (!sequence_of(a.seqs, token, q, bad)) {     // nobody's row: no weights, in case that its tile is somebody's
                for (size_t i = tid; i < 6 * a.ld / 16; i += T) reinterpret_cast<v4i*>(weights)[i] = v4i{0, 0, 0, 0};
                if (tid == 0) a.top[r] = 0;
                continue;
            }
            own = own_seen(a, q, token);
        }
        // weights are 0 up to where another row of the tile may see
        const uint32_t fill = min((uint32_t)a.ld, a.seqs.count ? a.prefix_cols + (own + 127) / 64 * 64 : a.prefix_cols);
        if (W > 1 && tid == 0) sh.any_top = 0;
        int64_t shift;
        bool top;
        if (!softmax_row<W, KIND, SUMS>(a.softmax, a.scores + (size_t)r * a.ld, weights, a.ld, Columns{a.prefix_len, a.prefix_cols, a.prefix_cols + own, own ? a.prefix_cols + own : a.prefix_len}, fill,
                                        live, power, sh, shift, top, bad)) {
            if (tid == 0) a.unsure[4 + atomicAdd(a.unsure, 1u)] = r;
            continue;
        }
        if (tid == 0 && a.shift_out) a.shift_out[((size_t)token * a.kv_heads + a.kv0 + r / rows) * a.group + (in - token * a.group)] = shift;
        const bool wave_top = __any(top);
        if constexpr (W == 1) {
            if (lane == 0) a.top[r] = wave_top;
        } else {
            if (wave_top && lane == 0) sh.any_top = 1;
            __syncthreads();
            if (tid == 0) a.top[r] = sh.any_top;
        }
    }
    raise(a.flag, bad);
}

// the products of five digits by three in an order that adds to no sum twice in a row
static constexpr int FIRST[15] = {0, 0, 0, 1, 2, 3, 4, 1, 1, 2, 3, 4, 2, 3, 4}, SECOND[15] = {0, 1, 2, 2, 2, 2, 2, 0, 1, 1, 1, 1, 0, 0, 0};
// What becomes of sums of weights times values: an output element, or a part's sum as its low 32 bits and, in units of 2^32, its size: twelve bytes, and the parts' sizes together
// say whether the whole fits
__device__ __forceinline__ void attn_finish(const AttnArgs& a, unsigned long long lo, int64_t size, uint32_t token, uint32_t head, uint32_t d, uint32_t& bad) {
    const int64_t v = (int64_t)lo;
    if (size > (3ll << 29) || size < -(3ll << 29) || v >= (1ll << 62) || v < -(1ll << 62)) { bad |= ZK_VALUES_RANGE; return; }
    auto q = [](int64_t x, const Divisor& s) { return s.shift >= 0 ? quotient<true>(x, s) : quotient<false>(x, s); };
    a.out[token * a.out_token + head * a.out_head + d] = narrow(q(q(v, a.sf_first), a.sf_second), bad);
}
template <int NS> __device__ __forceinline__ void attn_sum(const int32_t (&s)[NS], unsigned long long& lo, int64_t& size) {
    int64_t l = 0, h = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) l = l * 256 + s[i];
#pragma unroll
    for (int i = NS - 1; i >= 4; --i) h = h * 256 + s[i];
    lo = (unsigned long long)l + ((unsigned long long)h << 32);
    size = h + (l >> 32);
}
// Few rows: a wave takes 64 dimensions of 64 keys at a time; a lane reads four neighbouring dimensions of 16 keys, so that it has the 16 keys of a fragment of each.  weights: the lane's row and 16 keys of
// 64; keys from + 64 stream to end, 64 streams apart.  16000 keys of 8 heads of 128 24 us, 2.7 TB/s, bound by how much is on its way: two waves a SIMD, for
// which 62 registers are spilled (one wave with all of them: 29)
template <Heads HEADS> __device__ __forceinline__ void values_of(const AttnArgs& a, const Tile& t, uint32_t kv, uint32_t block, uint32_t first, uint32_t end, uint32_t stream, uint32_t streams, const int8_t* weights,
                                                              size_t ld, bool top, v4i (&acc)[9][4], uint32_t& bad) {
    const uint32_t lane = threadIdx.x & 63u, q = lane >> 4, d0 = block * 64 + 4 * (lane & 15u);
    if (first + stream * 64 >= end) return;
    const zk_i32_cache& cache = t.own ? a.own : a.prefix;
    const int32_t* values = (const int32_t*)cache.v + kv * cache.head_stride;
    const uint32_t sequence = t.own ? t.s.index : 0u;
    auto page = [&](uint32_t k) { return page_of(cache, sequence, min(k + lane, t.keys - 1)); };
    Page next = page(first + stream * 64);
    for (uint32_t k = first + stream * 64; k < end; k += 64 * streams) {
        const size_t mine = cache_at(cache, sequence, next, bad);
        next = page(k + 64 * streams);                     // looked up a step ahead
        v4i w[6];
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = *reinterpret_cast<const v4i*>(weights + i * ld + k);
        int32_t x[4][16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const v4i v = four_of<HEADS>(values + __shfl((unsigned long long)mine, (int)(q * 16 + i), 64), d0, a.dim);
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n][i] = v[n];
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            v4i v[4];
            digit_planes(x[n], v, bad);
            const bool four = __any(any_bits(v[3]));
#pragma unroll
            for (int i = 0; i < 15; ++i) acc[FIRST[i] + SECOND[i]][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[FIRST[i]], v[SECOND[i]], acc[FIRST[i] + SECOND[i]][n], 0, 0, 0);
            if (top)
#pragma unroll
                for (int j = 0; j < 3; ++j) acc[5 + j][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[5], v[j], acc[5 + j][n], 0, 0, 0);
            if (four)
#pragma unroll
                for (int i = 0; i < 6; ++i) acc[i + 3][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], v[3], acc[i + 3][n], 0, 0, 0);
        }
    }
}
// what 64 lanes have of the sums of 16 rows, added to sums [16][64 blocks of dimensions][2]: row 4 q + e, four dimensions
__device__ __forceinline__ void add_sums(unsigned long long* sums, uint32_t blocks, uint32_t block, const v4i (&acc)[9][4]) {
    const uint32_t lane = threadIdx.x & 63u, q = lane >> 4, d0 = block * 64 + 4 * (lane & 15u);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int32_t s[9];
#pragma unroll
            for (int i = 0; i < 9; ++i) s[i] = acc[i][n][e];
            unsigned long long lo;
            int64_t size;
            attn_sum<9>(s, lo, size);
            const uint32_t at = ((4 * q + e) * blocks * 64 + d0 + n) * 2;
            atomicAdd(&sums[at], lo);
            atomicAdd(&sums[at + 1], (unsigned long long)size);
        }
}
__device__ __forceinline__ void finish_tile(const AttnArgs& a, const Tile& t, uint32_t kv, const unsigned long long* sums, uint32_t blocks, uint32_t threads, uint32_t& bad) {
    for (uint32_t i = (t.lo - t.row0) * a.dim + threadIdx.x; i < (t.hi - t.row0) * a.dim; i += threads) {
        const uint32_t r = i / a.dim, d = i - r * a.dim, token = (t.row0 + r) / a.group, at = (r * blocks * 64 + d) * 2;
        attn_finish(a, sums[at], (int64_t)sums[at + 1], token, kv * a.group + (t.row0 + r - token * a.group), d, bad);
    }
}
template <Heads HEADS> __global__ void __launch_bounds__(256, 2) k_attn_values(const AttnArgs a, int own) {
    extern __shared__ unsigned long long sums64[];         // [16][64 blocks of dimensions][2]
    uint32_t bad = 0;
    Tile t;
    if (!tile_at<16>(a, own, blockIdx.z, t, bad)) { raise(a.flag, bad); return; }
    const uint32_t step = t.own ? a.own_step : a.prefix_step, first = blockIdx.y * step;
    if (first >= t.keys && !(a.direct && first == 0)) return;
    const uint32_t end = min(first + step, t.keys), blocks = (a.dim + 63) / 64, streams = 4 / blocks;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4, kv = a.kv0 + blockIdx.x, block = wave % blocks, stream = wave / blocks;
    const size_t row = (size_t)blockIdx.x * a.tokens * a.group + t.row0;
    for (uint32_t i = threadIdx.x; i < 16 * blocks * 64 * 2; i += 256) sums64[i] = 0;
    const uint32_t my_row = t.has(c) ? c : t.lo - t.row0;
    const bool top = __any(t.has(c) && a.top[row + my_row] != 0);
    v4i acc[9][4];
#pragma unroll
    for (int s = 0; s < 9; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[s][n] = v4i{0, 0, 0, 0};
    if (stream < streams) values_of<HEADS>(a, t, kv, block, first, end, stream, streams, a.weights + (row + my_row) * 6 * a.ld + t.col0 + q * 16, a.ld, top, acc, bad);
    __syncthreads();
    if (stream < streams) add_sums(sums64, blocks, block, acc);
    __syncthreads();
    if (!a.direct) {
        const size_t all = (size_t)a.heads_here * a.tokens * a.group;
        const size_t out = (((t.own ? a.prefix_splits : 0) + blockIdx.y) * all + row) * a.dim;
        for (uint32_t i = (t.lo - t.row0) * a.dim + threadIdx.x; i < (t.hi - t.row0) * a.dim; i += 256) {
            const uint32_t r = i / a.dim, at = (r * blocks * 64 + (i - r * a.dim)) * 2;
            a.parts_low[out + i] = (uint32_t)sums64[at];
            a.parts[out + i] = (int64_t)sums64[at + 1] + (uint32_t)((uint32_t)(sums64[at] >> 32) - (uint32_t)sums64[at + 1]);      // and what the waves' low halves carry
        }
    } else finish_tile(a, t, kv, sums64, blocks, 256, bad);
    raise(a.flag, bad);
}
// A tile of 16 rows with few keys, from scores to outputs in one launch: nothing leaves LDS between the steps.  One token of 32 heads over 200 keys 22 us (four launches: 29), the steps' latencies one after the
// other.  Up to 576 columns, what LDS holds of 16 rows, and 512 workgroups, two rounds of the units.  The sums of nine digits by four dimensions and the keys ahead are more than 256 registers: 55 to 106 are
// spilled for heads of up to 128 elements, 70 to 240 for longer ones, 448 to 638 where those are read element by element.
static constexpr uint32_t SMALL_COLS = 576, SMALL_LIVE = 4096;
template <int U, Heads HEADS, Weights KIND> __global__ void __launch_bounds__(512) k_attn_small(const AttnArgs a) {
    __shared__ __attribute__((aligned(16))) int64_t scores[16 * SMALL_COLS];
    __shared__ __attribute__((aligned(16))) int8_t weights[16][6 * SMALL_COLS];
    __shared__ int32_t live[KIND == Weights::SERIES ? SMALL_LIVE : 1];
    __shared__ double power[64];
    __shared__ RowShared<1> sh;
    __shared__ uint32_t tops[16];
    __shared__ v4i fourth[1][U][64];
    uint32_t bad = 0;
    Tile t;
    if (!tile_at<16>(a, a.seqs.count != 0, blockIdx.y, t, bad)) { raise(a.flag, bad); return; }
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4, kv = blockIdx.x, blocks = (a.dim + 63) / 64, streams = 8 / blocks, block = wave % blocks, stream = wave / blocks;
    Tile shared = t;                     // the same rows, the prefix's keys
    shared.own = false; shared.keys = a.prefix_len; shared.col0 = 0;
    softmax_tables<512, KIND>(a.softmax, live, power);
    if (a.prefix_len) scores_of<U, 1, HEADS, 8, false>(a, shared, kv, 0, a.prefix_len, fourth, scores, a.ld, bad);
    if (t.own && t.keys) scores_of<U, 1, HEADS, 8, false>(a, t, kv, 0, t.keys, fourth, scores + t.col0, a.ld, bad);
    __syncthreads();
    for (uint32_t r = wave; r < 16; r += 8) {
        bool top = false;
        if (t.has(r)) {
            const uint32_t token = (t.row0 + r) / a.group, own = t.own ? own_seen(a, t.s, token) : 0;
            int64_t shift;
            softmax_row<1, KIND, Sums::BOTH>(a.softmax, scores + r * a.ld, weights[r], a.ld, Columns{a.prefix_len, a.prefix_cols, a.prefix_cols + own, own ? a.prefix_cols + own : a.prefix_len}, (uint32_t)a.ld, live,
                                             power, sh, shift, top, bad);
            if (lane == 0 && a.shift_out) a.shift_out[((size_t)token * a.kv_heads + kv) * a.group + (t.row0 + r - token * a.group)] = shift;
        } else
            for (uint32_t i = lane; i < 6 * a.ld / 16; i += 64) reinterpret_cast<v4i*>(weights[r])[i] = v4i{0, 0, 0, 0};
        const bool any = __any(top);
        if (lane == 0) tops[r] = any;
    }
    __syncthreads();
    unsigned long long* sums = reinterpret_cast<unsigned long long*>(scores);      // the scores are used up
    for (uint32_t i = threadIdx.x; i < 16 * blocks * 64 * 2; i += 512) sums[i] = 0;
    const bool top = __any(tops[c] != 0);
    v4i acc[9][4];
#pragma unroll
    for (int s = 0; s < 9; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[s][n] = v4i{0, 0, 0, 0};
    if (stream < streams) {
        const int8_t* mine = weights[c] + q * 16;
        if (a.prefix_len) values_of<HEADS>(a, shared, kv, block, 0, a.prefix_len, stream, streams, mine, a.ld, top, acc, bad);
        if (t.own) values_of<HEADS>(a, t, kv, block, 0, t.keys, stream, streams, mine + t.col0, a.ld, top, acc, bad);
    }
    __syncthreads();
    if (stream < streams) add_sums(sums, blocks, block, acc);
    __syncthreads();
    finish_tile(a, t, kv, sums, blocks, 512, bad);
    raise(a.flag, bad);
}
// what a wave has of a tile's sums: 16 rows from row_in on by 64 dimensions from d0 on, of head z of the launch
__device__ __forceinline__ void tile_out(const AttnArgs& a, const Tile& t, int own, uint32_t kv, uint32_t z, size_t row, uint32_t row_in, uint32_t d0, const v4i (&acc)[9][4], uint32_t& bad) {
    typedef long long v2l __attribute__((ext_vector_type(2)));
    const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, q = lane >> 4, d = d0 + 4 * c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t at = row_in + 4 * q + e, in = t.row0 + at, token = in / a.group;
        if (!t.has(at) || d >= a.dim) continue;
        unsigned long long lo[4];
        int64_t size[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            int32_t s[9];
#pragma unroll
            for (int i = 0; i < 9; ++i) s[i] = acc[i][n][e];
            attn_sum<9>(s, lo[n], size[n]);
        }
        const size_t part = (((own ? a.prefix_splits : 0) + blockIdx.y) * ((size_t)a.heads_here * a.tokens * a.group) + row + at) * a.dim + d;
        if (!a.direct && a.dim % 4 == 0) {
            *reinterpret_cast<v4i*>(a.parts_low + part) = v4i{(int32_t)lo[0], (int32_t)lo[1], (int32_t)lo[2], (int32_t)lo[3]};
            *reinterpret_cast<v2l*>(a.parts + part) = v2l{size[0], size[1]};
            *reinterpret_cast<v2l*>(a.parts + part + 2) = v2l{size[2], size[3]};
            continue;
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (d + n >= a.dim) continue;
            if (!a.direct) {
                a.parts_low[part + n] = (uint32_t)lo[n];
                a.parts[part + n] = size[n];
            } else attn_finish(a, lo[n], size[n], token, kv * a.group + (in - token * a.group), d + n, bad);
        }
    }
}
// Many rows: 64 rows by 128 dimensions, a wave 16 by 64.  The workgroup splits 64 keys' values into digits together, the next ones while this step's are multiplied: a lane four keys of four
// dimensions, in LDS as fragments.  128 rows over 8192 keys of 8 heads of 128 46 us, 1.4 POP/s
template <Heads HEADS> __global__ void __launch_bounds__(512, 2) k_attn_values_tile(const AttnArgs a, int own) {
    __shared__ __attribute__((aligned(16))) int8_t planes[2][4][8][64][16], weight[2][4][6][64][16];      // fragments of the values and, [16 rows], of the weights
    __shared__ uint32_t wide[3];                           // of the step, the next and the one after that
    uint32_t bad = 0;
    Tile t;
    const uint32_t dim_blocks = (a.dim + 127) / 128, z = blockIdx.x / dim_blocks, dim0 = (blockIdx.x - z * dim_blocks) * 128;
    if (!tile_at<64>(a, own, blockIdx.z, t, bad)) { raise(a.flag, bad); return; }
    const uint32_t step = t.own ? a.own_step : a.prefix_step, first = blockIdx.y * step;
    if (first >= t.keys && !(a.direct && first == 0)) return;
    const uint32_t end = min(first + step, t.keys), steps = (end - first + 63) / 64;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4, kv = a.kv0 + z, row_in = (wave >> 1) * 16, block = wave & 1u;
    const size_t row = (size_t)z * a.tokens * a.group + t.row0;
    const zk_i32_cache& cache = t.own ? a.own : a.prefix;
    // a lane's share of the values: dimensions 4 dq .. 4 dq + 3 of keys 4 kq .. 4 kq + 3
    const uint32_t dq = threadIdx.x & 31u, kq = threadIdx.x >> 5, d0 = dim0 + 4 * dq;
    const int32_t* values = (const int32_t*)cache.v + kv * cache.head_stride;
    const uint32_t mine = t.has(row_in + c) ? row_in + c : t.lo - t.row0;
    const bool top = __any(a.top[row + mine] != 0);
    const int8_t* weights = a.weights + (row + mine) * 6 * a.ld + t.col0 + q * 16 + first;
    int32_t x[4][4];
    const uint32_t sequence = t.own ? t.s.index : 0u;
    auto page = [&](uint32_t i) { return page_of(cache, sequence, min(first + i * 64 + wave * 8 + (lane & 7u), t.keys - 1)); };
    Page next{0, 0};
    auto fetch = [&](uint32_t i) {
        const size_t at = cache_at(cache, sequence, next, bad);
        next = page(i + 1);                                // looked up a step ahead
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const v4i v = four_of<HEADS>(values + __shfl((unsigned long long)at, (int)((kq & 1u) * 4 + e), 64), d0, a.dim);
#pragma unroll
            for (int n = 0; n < 4; ++n) x[e][n] = v[n];
        }
    };
    // two waves have the same rows: each brings three digits of them to LDS
    auto fetch_weights = [&](uint32_t i) {
#pragma unroll
        for (int k = 0; k < 3; ++k) load_to_lds(weights + (block * 3 + k) * a.ld + i * 64, &weight[i & 1u][wave >> 1][block * 3 + k][0][0]);
    };
    auto split = [&](uint32_t i) {
        int32_t most = x[0][0];
        uint32_t upper = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            uint32_t d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                most = max(most, x[e][n]);
                d[e] = digit_bytes((uint32_t)x[e][n]);
                upper |= d[e];
            }
            const uint32_t f = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), g = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
            const uint32_t h = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), j = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
            const uint32_t p[4] = {__builtin_amdgcn_perm(h, f, 0x05040100u), __builtin_amdgcn_perm(h, f, 0x07060302u), __builtin_amdgcn_perm(j, g, 0x05040100u), __builtin_amdgcn_perm(j, g, 0x07060302u)};
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(&planes[i & 1u][k][(dq >> 4) * 4 + n][(kq >> 2) * 16 + (dq & 15u)][(kq & 3u) * 4]) = p[k];
        }
        bad |= most > 0x7F7F7F7F ? (uint32_t)ZK_VALUES_RANGE : 0u;
        if (upper >> 24) wide[i % 3] = 1;
    };
    v4i acc[9][4];
#pragma unroll
    for (int s = 0; s < 9; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[s][n] = v4i{0, 0, 0, 0};
    if (threadIdx.x < 3) wide[threadIdx.x] = 0;
    __syncthreads();
    if (steps) {
        next = page(0);
        fetch(0);
        fetch_weights(0);
        split(0);
    }
    __syncthreads();
    for (uint32_t i = 0; i < steps; ++i) {
        v4i w[6];
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = *reinterpret_cast<const v4i*>(&weight[i & 1u][wave >> 1][k][lane][0]);
        if (i + 1 < steps) {
            fetch(i + 1);
            fetch_weights(i + 1);
        }
        if (threadIdx.x == 0) wide[(i + 2) % 3] = 0;       // read last in the step before, written next in the step behind
        const bool four = wide[i % 3] != 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            v4i v[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) v[j] = *reinterpret_cast<const v4i*>(&planes[i & 1u][j][block * 4 + n][lane][0]);
#pragma unroll
            for (int e = 0; e < 15; ++e) acc[FIRST[e] + SECOND[e]][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[FIRST[e]], v[SECOND[e]], acc[FIRST[e] + SECOND[e]][n], 0, 0, 0);
            if (top)
#pragma unroll
                for (int j = 0; j < 3; ++j) acc[5 + j][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[5], v[j], acc[5 + j][n], 0, 0, 0);
            if (four) {
                const v4i u = *reinterpret_cast<const v4i*>(&planes[i & 1u][3][block * 4 + n][lane][0]);
#pragma unroll
                for (int k = 0; k < 6; ++k) acc[k + 3][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[k], u, acc[k + 3][n], 0, 0, 0);
            }
        }
        if (i + 1 < steps) split(i + 1);
        __syncthreads();
    }
    tile_out(a, t, own, kv, z, row, row_in, dim0 + block * 64, acc, bad);
    raise(a.flag, bad);
}
// The same where the values have been split already (k_attn_split): their fragments and the weights' go straight to LDS, two steps ahead.  2048 rows over 2048 keys of 8 heads of
// 128 72 us, 1.8 POP/s (splitting in every tile: 99); the barrier that every step of 60 matrix instructions a wave ends with bounds it
__global__ void __launch_bounds__(512, 2) k_attn_values_split(const AttnArgs a, int own) {
    // a variable a buffer: the compiler waits for a direct load before every read of the variable that it writes
    typedef int8_t Values[3][8][1024];                     // [digit][16 dimensions]
    typedef int8_t WeightsOf[4][6][1024];                  // [16 rows][digit]
    __shared__ __attribute__((aligned(16))) Values v0, v1, v2;
    __shared__ __attribute__((aligned(16))) WeightsOf w0, w1, w2;
    constexpr int LOADS = 6;
    uint32_t bad = 0;
    Tile t;
    const uint32_t dim_blocks = (a.dim + 127) / 128, z = blockIdx.x / dim_blocks, dim0 = (blockIdx.x - z * dim_blocks) * 128;
    if (!tile_at<64>(a, own, blockIdx.z, t, bad)) { raise(a.flag, bad); return; }
    const uint32_t step = t.own ? a.own_step : a.prefix_step, first = blockIdx.y * step;
    if (first >= t.keys && !(a.direct && first == 0)) return;
    const uint32_t end = min(first + step, t.keys), steps = (end - first + 63) / 64;
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = lane & 15u, q = lane >> 4, kv = a.kv0 + z, row_in = (wave >> 1) * 16, block = wave & 1u;
    const size_t row = (size_t)z * a.tokens * a.group + t.row0;
    const uint32_t mine = t.has(row_in + c) ? row_in + c : t.lo - t.row0, quads = (a.dim + 63) / 64 * 4, tiles = a.split_tiles[t.own] / 4;
    const bool top = __any(a.top[row + mine] != 0);
    const int8_t* weights = a.weights + (row + mine) * 6 * a.ld + t.col0 + q * 16 + first;
    const SplitPart& part = a.split[t.own];
    // a wave brings one of the eight tiles of 16 dimensions, where there are that many, and three digits of its 16 rows
    const size_t block0 = (size_t)z * tiles + first / 64;
    const uint32_t my_tile = min(dim0 / 16 + wave, quads - 1);
    auto fetch = [&](uint32_t i, Values& v, WeightsOf& w) {
        i = min(i, steps - 1);                             // behind the last step that again: never multiplied
        const int8_t* from = part.v + ((block0 + i) * quads + my_tile) * 4096 + lane * 16;
#pragma unroll
        for (int k = 0; k < 3; ++k) load_to_lds(from + k * 1024, &v[k][wave][0]);
#pragma unroll
        for (int k = 0; k < 3; ++k) load_to_lds(weights + (block * 3 + k) * a.ld + i * 64, &w[wave >> 1][block * 3 + k][0]);
    };
    // steps with a fourth digit, 128 of them at most: asked for one by one, the answers would wait for the loads behind them
    static_assert(MOST_STEP <= 128 * 64, "two words of steps");
    const unsigned long long wide[2] = {__ballot(lane < steps && part.v_wide[block0 + min(lane, steps - 1)] != 0), __ballot(lane + 64 < steps && part.v_wide[block0 + min(lane + 64, steps - 1)] != 0)};
    v4i acc[9][4];
#pragma unroll
    for (int s = 0; s < 9; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[s][n] = v4i{0, 0, 0, 0};
    // A step's pieces are in LDS when of every wave's loads only those of the next step are on their way, and all waves are past the barrier; the buffer read last is free then
    auto arrived = [&] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(LOADS | 7 << 4);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](uint32_t i, const Values& v, const WeightsOf& w) {
        if (i >= steps) return;
        v4i x[6];
#pragma unroll
        for (int k = 0; k < 6; ++k) x[k] = *reinterpret_cast<const v4i*>(&w[wave >> 1][k][lane * 16]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            v4i y[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) y[j] = *reinterpret_cast<const v4i*>(&v[j][block * 4 + n][lane * 16]);
#pragma unroll
            for (int e = 0; e < 15; ++e) acc[FIRST[e] + SECOND[e]][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[FIRST[e]], y[SECOND[e]], acc[FIRST[e] + SECOND[e]][n], 0, 0, 0);
            if (top)
#pragma unroll
                for (int j = 0; j < 3; ++j) acc[5 + j][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[5], y[j], acc[5 + j][n], 0, 0, 0);
        }
        if ((i < 64 ? wide[0] >> i : wide[1] >> (i - 64)) & 1u)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const v4i u = *reinterpret_cast<const v4i*>(part.v + (((block0 + i) * quads + min(dim0 / 16 + block * 4 + n, quads - 1)) * 4 + 3) * 1024 + lane * 16);
#pragma unroll
                for (int k = 0; k < 6; ++k) acc[k + 3][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[k], u, acc[k + 3][n], 0, 0, 0);
            }
    };
    if (steps) {
        fetch(0, v0, w0);
        fetch(1, v1, w1);
        for (uint32_t i = 0; i < steps; i += 3) {
            arrived(); fetch(i + 2, v2, w2); multiply(i, v0, w0);
            arrived(); fetch(i + 3, v0, w0); multiply(i + 1, v1, w1);
            arrived(); fetch(i + 4, v1, w1); multiply(i + 2, v2, w2);
        }
        __builtin_amdgcn_s_waitcnt(7 << 4 | 15 << 8);      // vmcnt 0: no load into LDS outlives the workgroup
    }
    tile_out(a, t, own, kv, z, row, row_in, dim0 + block * 64, acc, bad);
    raise(a.flag, bad);
}
// The parts' sums added up, 64 outputs a workgroup, by four shares of the parts or, where outputs are few, sixteen; rows that see no key.  1024 rows of 128, 33 parts:
// 15 us, 3.5 TB/s (parts of sixteen bytes: 20)
__global__ void __launch_bounds__(1024) k_attn_join(const AttnArgs a) {
    __shared__ unsigned long long sums[16][64][2];
    const uint32_t share = threadIdx.x >> 6, shares = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const size_t id = (size_t)blockIdx.x * 64 + lane, rows = (size_t)a.tokens * a.group, all = a.heads_here * rows;
    const bool inside = id < all * a.dim;
    const uint32_t r = inside ? (uint32_t)(id / a.dim) : 0, d = (uint32_t)(id - (size_t)r * a.dim), kv = (uint32_t)(r / rows), in = (uint32_t)(r - kv * rows), token = in / a.group;
    uint32_t bad = 0, own = 0;
    bool has = inside;
    if (a.seqs.count && inside) {
        Sequence s;
        has = sequence_of(a.seqs, token, s, bad);
        if (has) own = (own_seen(a, s, token) + a.own_step - 1) / a.own_step;
    }
    unsigned long long lo = 0, size = 0;
    if (has) {
        const uint32_t parts = a.prefix_splits + own;
        const size_t at = (size_t)r * a.dim + d;
#pragma unroll 4
        for (uint32_t i = share; i < parts; i += shares) {
            lo += a.parts_low[i * all * a.dim + at];
            size += (unsigned long long)a.parts[i * all * a.dim + at];
        }
        lo += size << 32;
    }
    sums[share][lane][0] = lo;
    sums[share][lane][1] = size;
    __syncthreads();
    if (has && share == 0) {
        for (uint32_t i = 1; i < shares; ++i) { lo += sums[i][lane][0]; size += sums[i][lane][1]; }
        attn_finish(a, lo, (int64_t)size, token, (a.kv0 + kv) * a.group + (in - token * a.group), d, bad);
    }
    raise(a.flag, bad);
}

// ---- logits -------------------------------------------------------------------------------------------------------------------------------
static constexpr int32_t NO_TOKEN = INT32_MIN;
static constexpr uint32_t LOGITS_THREADS = 512, LOGITS_SPAN = 4096;      // a workgroup's lanes and tokens
struct TokenLists { const int32_t *tokens, *values, *starts; uint32_t total; };      // row r's: starts[r] .. starts[r + 1]
struct LogitsArgs {
    int32_t *out, *token;
    const int32_t* logits;
    size_t ld_out, ld;
    uint32_t rows, vocab, spans;
    TokenLists history, bias;
    const int32_t* penalties;            // a row's: repeated, by count, once
    const uint32_t* mask;
    size_t ld_mask;
    uint32_t mask_rows;
    Divisor sf;
    unsigned long long* best;            // [row][span]
    uint32_t* flag;
};
__device__ __forceinline__ bool list_of(const TokenLists& l, uint32_t row, uint32_t& from, uint32_t& to, uint32_t& bad) {
    if (!l.starts) return false;
    const int32_t f = l.starts[row], t = l.starts[row + 1];
    if (f < 0 || t < f || (uint32_t)t > l.total) { bad |= ZK_VALUES_POSITION; return false; }
    from = (uint32_t)f; to = (uint32_t)t;
    return true;
}
// larger values first, among equals the lower token; 0: none
__device__ __forceinline__ unsigned long long choice(int32_t value, uint32_t token) { return value == NO_TOKEN ? 0ull : (unsigned long long)((uint32_t)value ^ 0x80000000u) << 32 | (0xFFFFFFFFu - token); }
__device__ __forceinline__ int32_t chosen(unsigned long long best) { return best ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : -1; }
__device__ __forceinline__ unsigned long long block_best(unsigned long long best, unsigned long long* of_wave) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) best = max(best, (unsigned long long)__shfl_xor(best, off, 64));
    if ((threadIdx.x & 63u) == 0) of_wave[threadIdx.x >> 6] = best;
    __syncthreads();
    best = 0;
    for (uint32_t i = 0; i < blockDim.x / 64; ++i) best = max(best, of_wave[i]);
    return best;
}
// A workgroup takes a stretch of a row, eight tokens a lane.  Its logits and mask are on their way while it reads the row's lists, eight entries a lane at a time, and counts and adds up in LDS what
// falls into the stretch.  BIAS: there are biases.  Issue bounds it: 64 rows of 128257 with 8000 tokens of history each 29 us, 2.3 TB/s, of which every stretch's way through the row's list
// is half; one row of 32000 4.9 us, latency.
template <bool POW2, bool BIAS> __global__ void __launch_bounds__(LOGITS_THREADS) k_logits(const LogitsArgs a) {
    constexpr int N = 8, T = LOGITS_THREADS;
    static_assert(LOGITS_SPAN == N * T, "a stretch is eight tokens a lane");
    __shared__ uint32_t count[LOGITS_SPAN];
    __shared__ unsigned long long add[BIAS ? LOGITS_SPAN : 1];
    __shared__ unsigned long long of_wave[LOGITS_THREADS / 64];
    const uint32_t row = blockIdx.y, first = blockIdx.x * LOGITS_SPAN, n = min(LOGITS_SPAN, a.vocab - first);
    uint32_t bad = 0, from = 0, to = 0;
    const uint32_t* mask = a.mask ? a.mask + (a.mask_rows == 1 ? 0 : row) * a.ld_mask : nullptr;
    const int32_t* in = a.logits + row * a.ld + first;
    int32_t l[N];
    uint32_t bits[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {                          // beyond the stretch its last
        const uint32_t i = min(threadIdx.x + e * T, n - 1);
        l[e] = in[i];
        bits[e] = mask ? mask[(first + i) >> 5] : 0xFFFFFFFFu;
    }
    for (uint32_t i = threadIdx.x * 4; i < LOGITS_SPAN; i += T * 4) {
        *reinterpret_cast<v4i*>(&count[i]) = v4i{0, 0, 0, 0};
        if constexpr (BIAS) {
            *reinterpret_cast<v4i*>(&add[i]) = v4i{0, 0, 0, 0};
            *reinterpret_cast<v4i*>(&add[i + 2]) = v4i{0, 0, 0, 0};
        }
    }
    __syncthreads();
    auto list = [&](const TokenLists& lists, auto put) {
        if (!list_of(lists, row, from, to, bad)) return;
        for (uint32_t i0 = from + threadIdx.x; i0 < to; i0 += T * N) {
            uint32_t token[N];
#pragma unroll
            for (int e = 0; e < N; ++e) token[e] = (uint32_t)lists.tokens[min(i0 + e * T, to - 1)];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const uint32_t i = i0 + e * T;
                if (i >= to) continue;
                bad |= token[e] >= a.vocab ? (uint32_t)ZK_VALUES_POSITION : 0u;
                if (token[e] - first < n) put(token[e] - first, i);
            }
        }
    };
    list(a.history, [&](uint32_t at, uint32_t) { atomicAdd(&count[at], 1u); });
    if constexpr (BIAS) list(a.bias, [&](uint32_t at, uint32_t i) { atomicAdd(&add[at], (unsigned long long)(int64_t)a.bias.values[i]); });
    __syncthreads();
    int32_t repeat = 0, frequency = 0, presence = 0;
    if (a.penalties) {
        repeat = a.penalties[3 * (size_t)row]; frequency = a.penalties[3 * (size_t)row + 1]; presence = a.penalties[3 * (size_t)row + 2];
        if (repeat <= 0) { bad |= ZK_VALUES_RANGE; repeat = 1; }
    }
    const Divisor by_repeat{repeat, repeat >> 1, 1.0 / (double)repeat, -1};
    int32_t most = NO_TOKEN;
    uint32_t most_at = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t i = threadIdx.x + e * T;
        if (i >= n) continue;
        const uint32_t token = first + i, c = count[i];
        if ((bits[e] >> (token & 31u) & 1u) == 0) l[e] = NO_TOKEN;
        bool changed = c != 0;
        if constexpr (BIAS) changed |= add[i] != 0;
        if (changed && l[e] != NO_TOKEN) {
            int64_t v = l[e];
            if (c != 0 && a.penalties) {
                if (v > 0) v = quotient_general(v * a.sf.s, by_repeat);
                else v = quotient<POW2>(v * repeat, a.sf);
                v = narrow(v, bad);
                v -= narrow((int64_t)frequency * c + presence, bad);
            }
            if constexpr (BIAS) v += narrow((int64_t)add[i], bad);
            l[e] = narrow(v, bad);
            if (l[e] == NO_TOKEN) bad |= ZK_VALUES_RANGE;
        }
        if (a.out) a.out[row * a.ld_out + token] = l[e];
        if (l[e] > most) { most = l[e]; most_at = token; }             // tokens ascend: the first of equals
    }
    if (a.token) {
        const unsigned long long best = block_best(choice(most, most_at), of_wave);
        if (threadIdx.x == 0) {
            if (a.spans == 1) a.token[row] = chosen(best);
            else a.best[(size_t)row * a.spans + blockIdx.x] = best;
        }
    }
    raise(a.flag, bad);
}
__global__ void __launch_bounds__(64) k_logits_best(int32_t* __restrict__ token, const unsigned long long* __restrict__ best, uint32_t spans) {
    __shared__ unsigned long long of_wave[1];
    unsigned long long b = 0;
    for (uint32_t i = threadIdx.x; i < spans; i += 64) b = max(b, best[(size_t)blockIdx.x * spans + i]);
    b = block_best(b, of_wave);
    if (threadIdx.x == 0) token[blockIdx.x] = chosen(b);
}

// ---- entry points -----------------------------------------------------------------------------------------------------------------------------------
static int check_cache(const zk_i32_cache* c, const char* name, uint32_t sequences, uint32_t most, uint32_t heads, uint32_t dim) {
    ZK_ARG(c->k != nullptr && c->v != nullptr, std::string(name) + ": a cache without keys or values");
    ZK_ARG(c->page_size > 0 && c->pages > 0, std::string(name) + ": a cache without pages");
    ZK_ARG(c->page_table != nullptr ? (uint64_t)c->table_cols * c->page_size >= most : c->page_size >= most && c->pages >= sequences,
           std::string(name) + ": a cache with fewer places than sequences or tokens");
    ZK_ARG((c->page_size == 1 || c->token_stride >= dim) && (heads == 1 || c->head_stride >= dim), std::string(name) + ": a cache whose heads overlap (a stride below the head's width)");
    const unsigned __int128 of_heads = (unsigned __int128)(heads - 1) * c->head_stride + dim, of_tokens = (unsigned __int128)(c->page_size - 1) * c->token_stride + dim;
    ZK_ARG(heads == 1 || c->page_size == 1 || c->token_stride >= of_heads || c->head_stride >= of_tokens, std::string(name) + ": a cache whose heads overlap");
    const unsigned __int128 page = (unsigned __int128)(heads - 1) * c->head_stride + (unsigned __int128)(c->page_size - 1) * c->token_stride + dim;
    ZK_ARG(c->pages == 1 || c->page_stride >= page || (heads > 1 && c->head_stride >= (unsigned __int128)(c->pages - 1) * c->page_stride + of_tokens && c->page_stride >= of_tokens),
           std::string(name) + ": a cache whose pages overlap");
    return 0;
}
static bool cache_aligned(const zk_i32_cache* c) { return ((c->page_stride | c->token_stride | c->head_stride) & 3) == 0 && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0; }

// How an attention call is cut: as many heads of keys at a time as keep scores and weights within 512 MB (fewer gain nothing), and its keys into parts, so that there are some 1024 workgroups (512 where rows are many)
struct AttnPlan { bool small, prefix64, own64, direct; uint32_t prefix_tiles, own_tiles, prefix_splits, prefix_step, own_splits, own_step, heads; size_t prefix_cols, cols, scores, weights, top, unsure, parts_high, parts, split_each; bool split[2]; uint32_t split_tiles[2]; };      // split_each: a head's
// From so many rows of a head of keys on its keys and values are split once for all of them. 8 heads of 128: at 128 rows over 8192 keys the split, scores and values take 25 + 35 + 53 us, tiles that each split
// what they read 41 + 46; at 2048 rows over as many keys 12 + 68 + 72 against 97 + 99
static constexpr size_t SPLIT_ROWS_FROM = 256;
static uint32_t split_dims(uint32_t dim) { return dim > 128 ? 256 : (dim + 63) / 64 * 64; }
static void attn_sizes(AttnPlan& p, uint32_t heads, size_t rows, uint32_t dim) {      // for that many heads of keys at a time
    auto round = [](size_t b) { return (b + 15) / 16 * 16; };
    p.heads = heads;
    p.scores = heads * rows * p.cols * 8;
    p.weights = heads * rows * p.cols * 6;
    p.top = round(heads * rows * 4);
    p.unsure = 16 + p.top;
    p.parts_high = round(heads * rows * (size_t)(p.direct ? 0 : p.prefix_splits + p.own_splits) * dim * 8);
    p.parts = round(p.parts_high + p.parts_high / 2);
}
static size_t attn_bytes(const AttnPlan& p) { return p.scores + p.weights + p.top + p.unsure + p.parts + p.heads * p.split_each; }
// room: the workspace.  Where it has none for the plan that is fastest, fewer heads go at a time; where it has none for one head either, nothing is split before and keys are cut as little as sums in 32 bits
// let them: what one head needs then grows with each of the call's sizes, so that a workspace for a larger call has room for it.
static AttnPlan attn_plan(uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t prefix_len, uint32_t sequences, uint32_t max_length, size_t room) {
    AttnPlan p{};
    const uint32_t group = heads / kv_heads;
    const size_t rows = (size_t)tokens * group;
    p.prefix_cols = ((size_t)prefix_len + 63) / 64 * 64;
    p.cols = p.prefix_cols + ((size_t)max_length + 63) / 64 * 64;
    const size_t small_tiles = sequences ? rows / 16 + sequences : cdiv(rows, 16);
    p.small = p.cols == 0 || (p.cols <= SMALL_COLS && small_tiles * kv_heads <= 512);
    if (p.small) { p.own_tiles = (uint32_t)small_tiles; p.heads = kv_heads; return p; }
    p.prefix64 = rows > 16;
    p.own64 = sequences && rows / sequences > 32;
    p.prefix_tiles = prefix_len ? cdiv(rows, p.prefix64 ? 64 : 16) : 0;
    p.own_tiles = sequences ? (uint32_t)(rows / (p.own64 ? 64 : 16)) + sequences : 0;
    auto cut = [&](uint32_t keys, size_t tiles, bool many, uint32_t& splits, uint32_t& step) {
        const size_t want = std::max<size_t>(1, (many ? 512 : 1024) / std::max<size_t>(1, tiles * kv_heads));
        splits = (uint32_t)std::min<size_t>(want, cdiv(keys, 256));
        splits = std::max(splits, cdiv(keys, MOST_STEP));
        step = splits ? (uint32_t)((cdiv(keys, splits) + 63) / 64 * 64) : 64;
        splits = cdiv(keys, step);
    };
    cut(prefix_len, p.prefix_tiles, p.prefix64, p.prefix_splits, p.prefix_step);
    cut(sequences ? max_length : 0, p.own_tiles, p.own64, p.own_splits, p.own_step);
    p.direct = p.prefix_splits + p.own_splits == 1;
    auto part = [&](bool many, uint32_t keys, int i) {
        p.split[i] = many && keys && rows >= SPLIT_ROWS_FROM && keys <= 65535u * 64;      // a grid's second side
        p.split_tiles[i] = p.split[i] ? cdiv(keys, 64) * 4 : 0;
    };
    part(p.prefix64, prefix_len, 0);
    part(p.own64 && sequences == 1, max_length, 1);
    p.split_each = (size_t)(p.split_tiles[0] + p.split_tiles[1]) * ((size_t)split_dims(dim) * 128 + 16);
    attn_sizes(p, 1, rows, dim);
    uint32_t most = (uint32_t)std::max<size_t>(1, std::min<size_t>(kv_heads, ((size_t)512 << 20) / std::max<size_t>(attn_bytes(p), 1)));
    if (most < kv_heads && p.own64 && p.own_splits == 1) {      // as many as fill the compute units evenly, one workgroup each
        auto used = [&](uint32_t h) { const size_t w = rows / 64 * h * cdiv(dim, 128); return w ? (double)w / (cdiv(w, 256) * 256.0) : 0.0; };
        for (uint32_t h = most; h >= std::max(1u, most / 2); --h) if (used(h) > used(most) + 0.02) most = h;
    }
    auto fit = [&] {
        for (uint32_t h = most; h >= 1; --h) {
            attn_sizes(p, h, rows, dim);
            if (attn_bytes(p) <= room) return true;
        }
        return false;
    };
    if (fit()) return p;
    auto cut_least = [&](uint32_t keys, uint32_t& splits, uint32_t& step) {
        step = std::min(MOST_STEP, std::max(64u, cdiv(keys, 64) * 64));
        splits = cdiv(keys, step);
    };
    cut_least(prefix_len, p.prefix_splits, p.prefix_step);
    cut_least(sequences ? max_length : 0, p.own_splits, p.own_step);
    p.direct = p.prefix_splits + p.own_splits == 1;
    p.split[0] = p.split[1] = false;
    p.split_tiles[0] = p.split_tiles[1] = 0;
    p.split_each = 0;
    (void)fit();
    return p;
}

extern "C" {

int zk_i32_cache_append(const zk_i32_cache* cache, const void* k, size_t k_token, size_t k_head, const void* v, size_t v_token, size_t v_head, uint32_t tokens, uint32_t heads, uint32_t dim,
                        uint32_t sequences, const void* starts, const void* lengths, void* flag_dev, void* stv) {
    static const char* name = "zk_i32_cache_append";
    if (tokens == 0 || heads == 0) return 0;
    ZK_ARG(cache != nullptr && k != nullptr && v != nullptr && lengths != nullptr && sequences > 0 && dim > 0, std::string(name) + ": null argument, no sequences or empty heads");
    ZK_ARG(starts != nullptr || tokens % sequences == 0, std::string(name) + ": without starts the tokens must divide among the sequences");
    ZK_ARG((uint64_t)heads * dim <= (1u << 30), std::string(name) + ": more than 2^30 elements a token");
    if (const int rc = check_cache(cache, name, sequences, 1, heads, dim)) return rc;
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    const uint64_t most = cache->page_table ? (uint64_t)cache->table_cols * cache->page_size : cache->page_size;
    const AppendArgs a{*cache, (const int32_t*)k, (const int32_t*)v, k_token, k_head, v_token, v_head, heads, dim,
                       Sequences{(const int32_t*)starts, (const int32_t*)lengths, sequences, tokens, (uint32_t)std::min<uint64_t>(most, 0x7FFFFFFFu)}, flag.dev};
    if (dim % 4 == 0 && cache_aligned(cache) && ((k_token | k_head | v_token | v_head) & 3) == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0)
        hipLaunchKernelGGL(k_cache_append<4>, dim3(tokens), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_cache_append<1>, dim3(tokens), dim3(256), 0, st, a);
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}

int zk_i32_softmax_free(void* softmax) {
    SoftmaxPlan* s = (SoftmaxPlan*)softmax;
    if (!s) return 0;
    int rc = 0;
    if (s->memory) rc = pool_free(s->memory, nullptr);
    delete s;
    return rc;
}
int zk_i32_softmax_prepare(void** softmax, const uint32_t* bs, int K, int L, int M, double scaling_factor_in, const double* thetas, uint32_t dim, void* stv) {
    static const char* name = "zk_i32_softmax_prepare";
    hipStream_t st = (hipStream_t)stv;
    ZK_ARG(softmax != nullptr && bs != nullptr && thetas != nullptr && dim > 0, std::string(name) + ": null argument or empty heads");
    ZK_ARG(K >= 1 && K <= DIGITS && L >= 0 && M >= 0 && L + M < K, std::string(name) + ": 1 to 8 digits, and at least one of them between the lowest L and the highest M");
    ZK_ARG(scaling_factor_in >= 1 && scaling_factor_in * std::sqrt((double)dim) <= 9007199254740992.0, std::string(name) + ": the scaling factor must lie within 1 .. 2^53 / sqrt(dim)");
    if (const int rc = CallFlag::not_captured(st, name)) return rc;
    std::unique_ptr<SoftmaxPlan> s(new SoftmaxPlan);
    s->dim = dim;
    SoftmaxArgs& a = s->a;
    a = SoftmaxArgs{};
    a.scale = scaling_factor_in * std::sqrt((double)dim);
    a.scale_inv = 1.0 / a.scale;
    a.scale_64 = 64.0 / (a.scale * 0.69314718055994530942);
    a.drop = 1;
    a.n = K - L;
    unsigned __int128 reach = 1;
    double most = 1;
    size_t entries = 0;
    for (int i = 0; i < K; ++i) {
        ZK_ARG(bs[i] >= 1 && bs[i] <= (1u << 28), std::string(name) + ": a radix must lie within 1 .. 2^28");
        reach *= bs[i];
        ZK_ARG(reach <= ((unsigned __int128)1 << 63), std::string(name) + ": the radices' product is above 2^63");
        const bool p2 = (bs[i] & (bs[i] - 1)) == 0;
        s->pow2 = s->pow2 && p2;
        if (i < L) { a.drop *= bs[i]; a.drop_bits += 31 - __builtin_clz(bs[i]); }
        else {
            a.radix[i - L] = bs[i];
            a.bits[i - L] = 31 - __builtin_clz(bs[i]);
            if (i < K - M) {
                const double theta = thetas[i - L];
                ZK_ARG(theta > 0 && theta < 2147483647.0, std::string(name) + ": a factor of the exponentials must lie within 0 .. 2^31 - 1");
                most *= std::floor(theta + 1.0);
                entries += bs[i];
            }
        }
    }
    ZK_ARG(most < 140000000000000.0, std::string(name) + ": weights of 1.4e14 and more (six digits of eight bits)");
    if (const int rc = pool_alloc((void**)&s->memory, entries * 4, st)) return rc;
    double weight = 1;
    size_t at = 0;
    for (int i = 0; i < K; ++i) {
        if (i >= L && i < K - M) {
            a.table[i - L] = s->memory + at;
            at += bs[i];
            hipLaunchKernelGGL(k_softmax_table_i32, dim3(cdiv(bs[i], 256)), dim3(256), 0, st, s->memory + at - bs[i], zkd::log_det(thetas[i - L]), weight / a.scale, bs[i]);
        }
        weight *= bs[i];
    }
    const int below = a.drop_bits + a.bits[0], all = below + a.bits[1];
    if (s->pow2 && M == 0 && a.n == 2 && below < 32 && all >= 32 && all < 64) {
        const double w0 = (double)a.drop / a.scale, w1 = w0 * bs[L], z = w0 * bs[L], reach = std::log(thetas[1]) + 0.75;      // beyond exp(-reach) theta is below 0.5
        for (int i = 0; i < 5; ++i) a.series[i] = i ? a.series[i - 1] * -w0 / i : thetas[0];      // theta exp(-w0 digit)
        a.series[0] += 0.5;
        a.guard = thetas[0] * (z * z * z * z * z / 60.0 + 0x1p-46);
        a.live = (uint32_t)std::max(1.0, std::min<double>(reach / w1 + 2.0, bs[L + 1]));      // a factor whose exponentials all lie below 0.5: the first entry, 0 as well
        a.upper_end = 1u << (all - 32);
        // z: the layer's heads from 64 elements on; `guard` alone would let narrower ones in, which has not been measured
        s->series = z <= 0x1p-7 && a.guard < 0.01 && reach / w1 + 2.0 <= MOST_LIVE;
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = hipStreamSynchronize(st);      // calls on any stream may use the tables
    if (e != hipSuccess) { (void)pool_free(s->memory, st); return hip_fail(e, "k_softmax_table_i32", __FILE__, __LINE__); }
    *softmax = s.release();
    return 0;
}

size_t zk_i32_attention_workspace(uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t prefix_len, uint32_t sequences, uint32_t max_length) {
    if (tokens == 0 || kv_heads == 0 || heads < kv_heads) return 0;
    return attn_bytes(attn_plan(tokens, heads, kv_heads, dim, prefix_len, sequences, max_length, SIZE_MAX));
}
int zk_i32_attention(void* out, size_t out_token, size_t out_head, const void* q, size_t q_token, size_t q_head, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                     const void* softmax, const zk_i32_cache* prefix, uint32_t prefix_len, const zk_i32_cache* own, uint32_t sequences, const void* starts, const void* lengths, uint32_t max_length,
                     int causal, uint32_t sf_first, uint32_t sf_second, void* shift, void* workspace, size_t workspace_bytes, void* flag_dev, void* stv) {
    static const char* name = "zk_i32_attention";
    if (tokens == 0 || heads == 0) return 0;
    const SoftmaxPlan* s = (const SoftmaxPlan*)softmax;
    ZK_ARG(out != nullptr && q != nullptr && s != nullptr, std::string(name) + ": null argument");
    ZK_ARG(dim > 0 && dim <= 256, std::string(name) + ": heads of 1 to 256 elements");
    ZK_ARG(kv_heads > 0 && heads % kv_heads == 0, std::string(name) + ": the heads must divide among those of keys and values");
    ZK_ARG((uint64_t)tokens * (heads / kv_heads) <= (1u << 20) && heads <= 65535, std::string(name) + ": more than 2^20 queries for a head of keys in one call, or more than 65535 heads");
    ZK_ARG(prefix_len <= (1u << 24) && max_length <= (1u << 24), std::string(name) + ": more than 2^24 keys");
    ZK_ARG((prefix != nullptr && prefix_len > 0) || own != nullptr, std::string(name) + ": neither a prefix nor sequences of their own");
    ZK_ARG(prefix_len == 0 || prefix != nullptr, std::string(name) + ": no prefix");
    ZK_ARG(own == nullptr || (sequences > 0 && sequences <= tokens + 65536u && lengths != nullptr), std::string(name) + ": sequences need lengths");
    ZK_ARG(own != nullptr || max_length == 0, std::string(name) + ": own keys without a cache");
    ZK_ARG(own == nullptr || starts != nullptr || tokens % sequences == 0, std::string(name) + ": without starts the tokens must divide among the sequences");
    ZK_ARG(sf_first > 0 && sf_second > 0, std::string(name) + ": a scaling factor of 0");
    ZK_ARG(out != q || (out_token == q_token && out_head == q_head), std::string(name) + ": in place with other strides");
    ZK_ARG((tokens == 1 || out_token >= dim) && (heads == 1 || out_head >= dim), std::string(name) + ": heads overlap (a stride below the head's width)");
    {
        const unsigned __int128 of_heads = (unsigned __int128)(heads - 1) * out_head + dim, of_tokens = (unsigned __int128)(tokens - 1) * out_token + dim;
        ZK_ARG(tokens == 1 || heads == 1 || out_token >= of_heads || out_head >= of_tokens, std::string(name) + ": the output's heads overlap");
    }
    if (prefix_len) if (const int rc = check_cache(prefix, name, 1, prefix_len, kv_heads, dim)) return rc;
    if (own) if (const int rc = check_cache(own, name, sequences, max_length, kv_heads, dim)) return rc;
    if (!own) sequences = 0;
    const AttnPlan p = attn_plan(tokens, heads, kv_heads, dim, prefix_len, sequences, max_length, workspace ? workspace_bytes : SIZE_MAX);
    ZK_ARG(p.prefix_tiles <= 65535u && p.own_tiles <= 65535u && (uint64_t)p.heads * cdiv(dim, 128) <= 65535u, std::string(name) + ": more than 65535 tiles of queries");
    hipStream_t st = (hipStream_t)stv;
    const size_t bytes = attn_bytes(p);
    ZK_ARG(workspace == nullptr || workspace_bytes >= bytes, std::string(name) + ": the workspace is smaller than zk_i32_attention_workspace says, and than the call needs for one head of keys at a time");
    ZK_ARG(((uintptr_t)workspace & 15) == 0, std::string(name) + ": the workspace must begin at a multiple of 16 bytes");
    ZK_ARG(dim == s->dim, std::string(name) + ": the softmax was prepared for heads of another width");
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    std::unique_ptr<Scratch> scratch;
    if (!workspace && bytes) {
        if (const int rc = CallFlag::not_captured(st, name)) return rc;
        scratch.reset(new Scratch(bytes, st));
        if (scratch->rc) return scratch->rc;
        workspace = scratch->p;
    }
    AttnArgs a{};
    a.out = (int32_t*)out; a.q = (const int32_t*)q; a.out_token = out_token; a.out_head = out_head; a.q_token = q_token; a.q_head = q_head;
    a.group = heads / kv_heads; a.dim = dim; a.kv_heads = kv_heads; a.shift_out = (int64_t*)shift; a.softmax = s->a;
    if (prefix_len) a.prefix = *prefix;
    if (own) a.own = *own;
    a.prefix_len = prefix_len; a.prefix_cols = (uint32_t)p.prefix_cols;
    a.seqs = Sequences{own ? (const int32_t*)starts : nullptr, (const int32_t*)lengths, sequences, tokens, max_length};
    a.causal = causal; a.sf_first = divisor(sf_first); a.sf_second = divisor(sf_second);
    a.scores = (int64_t*)workspace; a.ld = p.cols; a.weights = (int8_t*)workspace + p.scores; a.top = (uint32_t*)(a.weights + p.weights);
    a.unsure = (uint32_t*)((char*)a.top + p.top); a.parts = (int64_t*)((char*)a.unsure + p.unsure); a.parts_low = (uint32_t*)((char*)a.parts + p.parts_high); a.direct = p.direct;
    {
        int8_t* at = (int8_t*)a.parts + p.parts;
        for (int i = 0; i < 2; ++i) {
            const size_t tiles = (size_t)p.heads * p.split_tiles[i], bytes_of = tiles * split_dims(dim) * 64;
            a.split_tiles[i] = p.split_tiles[i];
            a.split[i] = SplitPart{at, at + bytes_of, (uint32_t*)(at + 2 * bytes_of), (uint32_t*)(at + 2 * bytes_of) + tiles};
            at += 2 * bytes_of + tiles * 16;
        }
    }
    a.tokens = tokens; a.prefix_tiles = p.prefix_tiles; a.prefix_splits = p.prefix_splits; a.prefix_step = p.prefix_step; a.own_splits = p.own_splits; a.own_step = p.own_step;
    a.flag = flag.dev;
    const bool fours = dim % 4 == 0 && ((q_token | q_head) & 3) == 0 && ((uintptr_t)q & 15) == 0 && (!prefix_len || cache_aligned(prefix)) && (!own || cache_aligned(own));
    const unsigned blocks = cdiv(dim, 64);
    auto heads_of = [&](auto launch) {
        if (fours && (dim == 64 || dim == 128 || dim == 256)) launch(std::integral_constant<Heads, Heads::BLOCKS>());
        else if (fours) launch(std::integral_constant<Heads, Heads::FOURS>());
        else launch(std::integral_constant<Heads, Heads::ANY>());
    };
    if (p.small) {
        auto small = [&](auto u, auto kind) {
            constexpr int U = decltype(u)::value;
            constexpr Weights KIND = decltype(kind)::value;
            heads_of([&](auto h) { hipLaunchKernelGGL((k_attn_small<U, decltype(h)::value, KIND>), dim3(kv_heads, p.own_tiles), dim3(512), 0, st, a); });
        };
        auto of_kind = [&](auto kind) {
            if (blocks == 1) small(std::integral_constant<int, 1>(), kind);
            else if (blocks == 2) small(std::integral_constant<int, 2>(), kind);
            else small(std::integral_constant<int, 4>(), kind);
        };
        if (s->series && a.softmax.live <= SMALL_LIVE) of_kind(std::integral_constant<Weights, Weights::SERIES>());
        else if (s->pow2) of_kind(std::integral_constant<Weights, Weights::POW2>());
        else of_kind(std::integral_constant<Weights, Weights::ANY>());
        ZK_LAUNCH_CHECK();
        return flag.end(name);
    }
    for (a.kv0 = 0; a.kv0 < kv_heads; a.kv0 += p.heads) {
        a.heads_here = std::min(p.heads, kv_heads - a.kv0);
        const size_t rows = (size_t)a.heads_here * tokens * a.group;
        // the prefix's keys, then the sequences' own
        auto both = [&](auto f) {
            if (p.prefix_tiles) f(0, p.prefix64, p.prefix_tiles, prefix_len, p.prefix_splits);
            if (p.own_tiles && max_length) f(1, p.own64, p.own_tiles, max_length, p.own_splits);
        };
        both([&](int of_own, bool many, unsigned tiles, uint32_t keys, unsigned) {
            if (p.split[of_own]) heads_of([&](auto h) { hipLaunchKernelGGL(k_attn_split<decltype(h)::value>, dim3(a.heads_here, cdiv(keys, 64)), dim3(256), 0, st, a, of_own); });
            const unsigned rt = !many ? 1 : 4;
            if (many) tiles = of_own ? tokens * a.group / (16 * rt) + sequences : cdiv((size_t)tokens * a.group, 16 * rt);
            a.score_keys = 1024;                   // a workgroup's, where that still makes 512 workgroups
            while (a.score_keys > 64 && (size_t)cdiv(keys, a.score_keys) * tiles * a.heads_here < 512) a.score_keys /= 2;
            const dim3 grid(a.heads_here, cdiv(keys, a.score_keys), tiles);      // heads first: workgroups go to the eight dies in turn, and a die's L2 has a head's keys then
            auto scores = [&](auto u, auto rt) {
                constexpr int U = decltype(u)::value, RT = decltype(rt)::value;
                heads_of([&](auto h) {
                    if constexpr (RT > 1)
                        if (p.split[of_own]) { hipLaunchKernelGGL((k_attn_scores<U, RT, decltype(h)::value, true>), grid, dim3(256), 0, st, a, of_own); return; }
                    hipLaunchKernelGGL((k_attn_scores<U, RT, decltype(h)::value, false>), grid, dim3(256), 0, st, a, of_own);
                });
            };
            auto wide = [&](auto u) {
                if (many) scores(u, std::integral_constant<int, 4>());
                else scores(u, std::integral_constant<int, 1>());
            };
            if (blocks == 1) wide(std::integral_constant<int, 1>());
            else if (blocks == 2) wide(std::integral_constant<int, 2>());
            else wide(std::integral_constant<int, 4>());
        });
        auto softmax_rows = [&](auto kind) {
            constexpr Weights KIND = decltype(kind)::value;
            const size_t lds = KIND == Weights::SERIES ? s->a.live * 4 : 0;
            if (rows < 256) {
                if (p.cols <= 2048) hipLaunchKernelGGL((k_attn_softmax<4, KIND, Sums::BOTH>), dim3((unsigned)rows), dim3(256), lds, st, a);
                else hipLaunchKernelGGL((k_attn_softmax<8, KIND, Sums::BOTH>), dim3((unsigned)rows), dim3(512), lds, st, a);
                return;
            }
            if (p.cols <= 2048) hipLaunchKernelGGL((k_attn_softmax<1, KIND, Sums::NEAR>), dim3((unsigned)std::min<size_t>(cdiv(rows, 4), 1024)), dim3(256), lds, st, a);
            else hipLaunchKernelGGL((k_attn_softmax<4, KIND, Sums::NEAR>), dim3((unsigned)std::min<size_t>(rows, 1024)), dim3(256), lds, st, a);
            if (p.cols <= 2048) hipLaunchKernelGGL((k_attn_softmax<4, KIND, Sums::IN_ORDER>), dim3((unsigned)std::min<size_t>(rows, 512)), dim3(256), lds, st, a);
            else hipLaunchKernelGGL((k_attn_softmax<8, KIND, Sums::IN_ORDER>), dim3((unsigned)std::min<size_t>(rows, 512)), dim3(512), lds, st, a);
        };
        if (s->series) softmax_rows(std::integral_constant<Weights, Weights::SERIES>());
        else if (s->pow2) softmax_rows(std::integral_constant<Weights, Weights::POW2>());
        else softmax_rows(std::integral_constant<Weights, Weights::ANY>());
        both([&](int of_own, bool many, unsigned tiles, uint32_t, unsigned splits) {
            if (many) {
                const dim3 grid(a.heads_here * cdiv(dim, 128), splits, tiles);
                if (p.split[of_own]) hipLaunchKernelGGL(k_attn_values_split, grid, dim3(512), 0, st, a, of_own);
                else heads_of([&](auto h) { hipLaunchKernelGGL(k_attn_values_tile<decltype(h)::value>, grid, dim3(512), 0, st, a, of_own); });
            } else {
                const dim3 grid(a.heads_here, splits, tiles);
                const size_t lds = 16 * (size_t)blocks * 64 * 16;
                heads_of([&](auto h) { hipLaunchKernelGGL(k_attn_values<decltype(h)::value>, grid, dim3(256), lds, st, a, of_own); });
            }
        });
        if (!p.direct) hipLaunchKernelGGL(k_attn_join, dim3(cdiv(rows * dim, 64)), dim3(rows * dim < 65536 ? 1024 : 256), 0, st, a);
    }
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}

size_t zk_i32_logits_workspace(uint32_t rows, uint32_t vocab) {
    const size_t spans = cdiv(vocab, LOGITS_SPAN);
    return spans <= 1 ? 0 : rows * spans * sizeof(unsigned long long);
}
int zk_i32_logits(void* out, size_t ld_out, void* token, const void* logits, size_t ld, uint32_t rows, uint32_t vocab, const void* history, uint32_t history_len, const void* history_starts,
                  const void* penalties, const void* bias_tokens, const void* bias_values, uint32_t bias_len, const void* bias_starts, const void* mask, size_t ld_mask, uint32_t mask_rows, uint32_t sf,
                  void* workspace, size_t workspace_bytes, void* flag_dev, void* stv) {
    static const char* name = "zk_i32_logits";
    if (rows == 0) return 0;
    ZK_ARG(logits != nullptr && (out != nullptr || token != nullptr) && vocab > 0, std::string(name) + ": null logits, no output or no tokens");
    ZK_ARG(vocab <= (1u << 30) && rows <= 65535, std::string(name) + ": more than 2^30 tokens or 65535 rows");
    ZK_ARG(rows == 1 || (ld >= vocab && (out == nullptr || ld_out >= vocab)), std::string(name) + ": rows overlap (a leading dimension below the number of tokens)");
    ZK_ARG(out != logits || rows == 1 || ld_out == ld, std::string(name) + ": in place with another leading dimension");
    ZK_ARG(history_starts == nullptr || ((history != nullptr || history_len == 0) && penalties != nullptr), std::string(name) + ": a history needs its tokens and penalties");
    ZK_ARG(history_starts != nullptr || (history == nullptr && penalties == nullptr), std::string(name) + ": a history or penalties without starts");
    ZK_ARG(bias_starts == nullptr || (bias_tokens != nullptr && bias_values != nullptr) || bias_len == 0, std::string(name) + ": biases need their tokens and values");
    ZK_ARG(bias_starts != nullptr || (bias_tokens == nullptr && bias_values == nullptr), std::string(name) + ": biases without starts");
    ZK_ARG(history_len <= 0x7FFFFFFFu && bias_len <= 0x7FFFFFFFu, std::string(name) + ": a list of more than 2^31 - 1 tokens");
    ZK_ARG(mask == nullptr ? mask_rows == 0 : (mask_rows == 1 || (mask_rows == rows && ld_mask >= (vocab + 31) / 32)), std::string(name) + ": a mask has one row or a row for each of the logits'");
    ZK_ARG(sf > 0 && sf <= 0x7FFFFFFFu, std::string(name) + ": a scaling factor of 0 or of 2^31 and more");
    hipStream_t st = (hipStream_t)stv;
    const size_t bytes = token ? zk_i32_logits_workspace(rows, vocab) : 0;
    ZK_ARG(workspace == nullptr || workspace_bytes >= bytes, std::string(name) + ": the workspace is smaller than zk_i32_logits_workspace says");
    ZK_ARG(((uintptr_t)workspace & 15) == 0, std::string(name) + ": the workspace must begin at a multiple of 16 bytes");
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    std::unique_ptr<Scratch> scratch;
    if (!workspace && bytes) {
        if (const int rc = CallFlag::not_captured(st, name)) return rc;
        scratch.reset(new Scratch(bytes, st));
        if (scratch->rc) return scratch->rc;
        workspace = scratch->p;
    }
    const uint32_t spans = cdiv(vocab, LOGITS_SPAN);
    const LogitsArgs a{(int32_t*)out, (int32_t*)token, (const int32_t*)logits, ld_out, ld, rows, vocab, spans,
                       TokenLists{(const int32_t*)history, nullptr, (const int32_t*)history_starts, history_len},
                       TokenLists{(const int32_t*)bias_tokens, (const int32_t*)bias_values, (const int32_t*)bias_starts, bias_len}, (const int32_t*)penalties, (const uint32_t*)mask, ld_mask, mask_rows,
                       divisor(sf), (unsigned long long*)workspace, flag.dev};
    const bool bias = bias_starts != nullptr && bias_len > 0;
    if (a.sf.shift >= 0 && bias) hipLaunchKernelGGL((k_logits<true, true>), dim3(spans, rows), dim3(LOGITS_THREADS), 0, st, a);
    else if (a.sf.shift >= 0) hipLaunchKernelGGL((k_logits<true, false>), dim3(spans, rows), dim3(LOGITS_THREADS), 0, st, a);
    else if (bias) hipLaunchKernelGGL((k_logits<false, true>), dim3(spans, rows), dim3(LOGITS_THREADS), 0, st, a);
    else hipLaunchKernelGGL((k_logits<false, false>), dim3(spans, rows), dim3(LOGITS_THREADS), 0, st, a);
    if (token && spans > 1) hipLaunchKernelGGL(k_logits_best, dim3(rows), dim3(64), 0, st, (int32_t*)token, (const unsigned long long*)workspace, spans);
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}

}  // extern "C"
