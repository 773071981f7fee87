// A decoder layer's values in the prover's integers, for gfx950: what the blocks' forward passes compute (rmsnorm.cu:36-39, self-attn.cu:47-56,
// ffn.cu:61-81, skip-connection.cu:15-18, and the rotary positions of llama-self-attn.py:42-73) without the remainders, multiplicities and
// field elements that only their proofs read.  Tensors are int32 in fixed point; every result is a whole number and equals what
// the class layer's tensors hold.
//
//   quotient   Q(t; s) = floor((t + floor(s / 2)) / s), the rescaling of rescaling.cu:13-19
//   norm       N(v; w)_j = Q(Q(w_j r; s) v_j; s),  r = the nearest integer to scale / sqrt(mean((v / scale)^2) + eps)
//   residual   h = x + Q(res Q(gate N(b; post); s); s), n = N(h; w)
//   rotary     (x0, x1) -> (Q(c x0 - t x1; s), Q(t x0 + c x1; s)), c and t the table's cosine and sine of the token's position
//   linear     Q(x W; s)
//   gated      Q(act[Q(x G; s_g)] Q(x U; s_u); s_h)
//
// Values that leave int32, activations outside the table and positions outside theirs raise bits of a flag on the device; nothing is read
// or written out of range for them.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <type_traits>
#include "field.hpp"
#include "planes.hpp"
#include "rt.hpp"
#include "../../include/zkllm_hip.h"

using namespace zk;

// ---- quotients --------------------------------------------------------------------------------------------------------------------------
// shift >= 0: s is 2^shift, else any.  POW2 is a template argument where a kernel divides often.
struct Divisor { int64_t s, half; double inv; int shift; };
static Divisor divisor(uint32_t s) { return Divisor{(int64_t)s, (int64_t)(s >> 1), 1.0 / (double)s, (s & (s - 1)) == 0 ? 31 - __builtin_clz(s) : -1}; }
// floor((t + s / 2) / s) for |t| <= 2^62, by the divisor's double-precision inverse: the first quotient is off by no more than 3 2^-53 2^62 / s + 1, what
// it leaves is below s + 2^11 in magnitude and divided exactly up to one unit.  Some 30 instructions against some 100 of a 64-bit division.
__device__ __forceinline__ int64_t quotient_general(int64_t t, const Divisor& d) {
    const int64_t n = t + d.half;
    int64_t q = (int64_t)floor((double)n * d.inv);
    int64_t r = n - q * d.s;
    const int64_t more = (int64_t)floor((double)r * d.inv);
    q += more;
    r -= more * d.s;
    return q - (r < 0 ? 1 : 0) + (r >= d.s ? 1 : 0);
}
template <bool POW2> __device__ __forceinline__ int64_t quotient(int64_t t, const Divisor& d) {
    if constexpr (POW2) return (t + d.half) >> d.shift;
    else return quotient_general(t, d);
}
__device__ __forceinline__ int64_t quotient_any(int64_t t, const Divisor& d) { return d.shift >= 0 ? (t + d.half) >> d.shift : quotient_general(t, d); }
__device__ __forceinline__ int32_t narrow(int64_t v, uint32_t& bad) {
    bad |= (v != (int64_t)(int32_t)v) ? (uint32_t)ZK_VALUES_RANGE : 0u;
    return (int32_t)v;
}
__device__ __forceinline__ void raise(uint32_t* flag, uint32_t bad) { if (bad) atomicOr(flag, bad); }

// ---- norms with the residual stream -------------------------------------------------------------------------------------------------------
struct NormArgs {
    int32_t *h, *n, *rms_inv;
    const int32_t *x, *b, *post, *gate, *w;
    size_t ldx, ldb;
    uint32_t cols, rows_per_gate;
    int32_t res;
    double scale, eps;
    int scale_exact;          // the scale is a power of two: dividing by it rounds nothing
    Divisor sf;
    uint32_t* flag;
};
// a workgroup's sum of 64-bit terms and its largest 32-bit magnitude, in every lane
__device__ __forceinline__ void block_sum_max(unsigned long long& s, uint32_t& m, unsigned long long* red_s, uint32_t* red_m) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        s += __shfl_xor(s, off, 64);
        const uint32_t o = __shfl_xor(m, off, 64);
        m = o > m ? o : m;
    }
    const uint32_t waves = (blockDim.x + 63) / 64;
    __syncthreads();                           // the arrays' last use is over
    if ((threadIdx.x & 63u) == 0) { red_s[threadIdx.x >> 6] = s; red_m[threadIdx.x >> 6] = m; }
    __syncthreads();
    s = 0; m = 0;
    for (uint32_t i = 0; i < waves; ++i) { s += red_s[i]; m = red_m[i] > m ? red_m[i] : m; }
}
// Whether the sum of squares, s by addition modulo 2^64, stands for the double-precision sum in index order that the layer's proof is made with
// (zk_row_sumsq_f64): then no addition of that sum rounds, in whatever order.
__device__ __forceinline__ bool sum_is_exact(unsigned long long s, uint32_t m, const NormArgs& a) {
    return a.scale_exact && (double)m * (double)m * (double)a.cols < 9.2e18 && s <= (1ull << 53);
}
__device__ __forceinline__ int32_t rms_inverse(double sumsq, const NormArgs& a) {
    const double v = 1.0 / sqrt(sumsq / (double)a.cols + a.eps);
    return (int32_t)rint(v * a.scale);
}
template <bool POW2> __device__ __forceinline__ int32_t normed(int32_t w, int32_t r, int32_t v, const Divisor& sf, uint32_t& bad) {
    const int32_t g = narrow(quotient<POW2>((int64_t)w * r, sf), bad);
    return narrow(quotient<POW2>((int64_t)g * v, sf), bad);
}

// A workgroup a row; lanes own columns threadIdx.x, threadIdx.x + blockDim.x, ...; every pass reads the row again.  A lane writes only columns that
// it alone reads, so h and n may be x or b themselves.
template <bool POW2> __global__ void __launch_bounds__(256) k_residual_norm_long(const NormArgs a) {
    __shared__ unsigned long long red_s[4];
    __shared__ uint32_t red_m[4];
    __shared__ double term[256], total;
    const size_t row = blockIdx.x;
    const int32_t* x = a.x + row * a.ldx;
    const int32_t* b = a.b ? a.b + row * a.ldb : nullptr;
    const int32_t* gate = a.gate ? a.gate + row / a.rows_per_gate * a.cols : nullptr;
    int32_t* h = a.h ? a.h + row * a.cols : nullptr;
    uint32_t bad = 0;
    auto statistic = [&](auto get) {
        unsigned long long s = 0;
        uint32_t m = 0;
        for (uint32_t j = threadIdx.x; j < a.cols; j += 256) {
            const int64_t v = get(j);
            s += (unsigned long long)(v * v);
            const uint32_t mag = (uint32_t)(v < 0 ? -v : v);
            m = mag > m ? mag : m;
        }
        block_sum_max(s, m, red_s, red_m);
        if (sum_is_exact(s, m, a)) return rms_inverse((double)s / a.scale / a.scale, a);
        double acc = 0.0;                      // in index order, a stretch of 256 terms at a time
        for (uint32_t j0 = 0; j0 < a.cols; j0 += 256) {
            const uint32_t j = j0 + threadIdx.x;
            const double v = j < a.cols ? (double)get(j) / a.scale : 0.0;
            __syncthreads();
            term[threadIdx.x] = v * v;
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t cnt = a.cols - j0 < 256u ? a.cols - j0 : 256u;
                for (uint32_t q = 0; q < cnt; ++q) acc += term[q];
            }
        }
        if (threadIdx.x == 0) total = acc;
        __syncthreads();
        const double t = total;
        __syncthreads();
        return rms_inverse(t, a);
    };
    int32_t r_post = 0;
    if (b && a.post) r_post = statistic([&](uint32_t j) { return b[j]; });
    auto stream = [&](uint32_t j) {            // the residual stream with the block's output
        if (!b) return x[j];
        int32_t q = b[j];
        if (a.post) q = normed<POW2>(a.post[j], r_post, q, a.sf, bad);
        if (gate) q = narrow(quotient<POW2>((int64_t)gate[j] * q, a.sf), bad);
        return narrow((int64_t)x[j] + quotient<POW2>((int64_t)a.res * q, a.sf), bad);
    };
    if (h) for (uint32_t j = threadIdx.x; j < a.cols; j += 256) h[j] = stream(j);
    if (a.n || a.rms_inv) {
        auto get = [&](uint32_t j) { return h ? h[j] : stream(j); };
        const int32_t r = statistic(get);
        if (a.rms_inv && threadIdx.x == 0) a.rms_inv[row] = r;
        if (a.n) for (uint32_t j = threadIdx.x; j < a.cols; j += 256) a.n[row * a.cols + j] = normed<POW2>(a.w[j], r, get(j), a.sf, bad);
    }
    raise(a.flag, bad);
}

// ---- rotary positions ------------------------------------------------------------------------------------------------------------------------
struct RopeArgs {
    void* out;
    const void* x;
    size_t out_token, out_head, x_token, x_head;
    uint32_t tokens, heads, dim, rot;
    int neighbours;
    const int2* table;
    uint32_t table_rows;
    const int32_t* positions;
    uint32_t first;
    Divisor sf;
    uint32_t* flag;
};
// entries beyond 2^30, the largest scale: two products of theirs could leave 64 bits
__device__ __forceinline__ int2 angle(int2 cs, uint32_t& bad) {
    const int32_t most = 1 << 30;
    if (cs.x > most || cs.x < -most || cs.y > most || cs.y < -most) { bad |= ZK_VALUES_RANGE; return make_int2(0, 0); }
    return cs;
}
__device__ __forceinline__ int64_t rope_get(const int32_t* p, uint32_t&) { return *p; }
__device__ __forceinline__ int64_t rope_get(const Fr* p, uint32_t& bad) {
    const Fr e = *p;
    const int64_t v = fr_to_i64(e);
    // an element that is no 32-bit integer: fr_to_i64 gives 0 for what does not fit 64 bits, and zero is told apart by its limbs
    const bool zero = !(e.v[0] | e.v[1] | e.v[2] | e.v[3] | e.v[4] | e.v[5] | e.v[6] | e.v[7]);
    if (v != (int64_t)(int32_t)v || (v == 0 && !zero)) { bad |= ZK_VALUES_RANGE; return 0; }
    return v;
}
__device__ __forceinline__ void rope_put(int32_t* p, int64_t v, uint32_t& bad) { *p = narrow(v, bad); }
__device__ __forceinline__ void rope_put(Fr* p, int64_t v, uint32_t&) { *p = fr_from_i64(v); }
// a lane a pair of the rotated part or an element of the rest
template <typename T, bool POW2> __global__ void __launch_bounds__(256) k_rope(const RopeArgs a, uint64_t base, uint64_t end) {
    const uint64_t id = base + (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= end) return;
    const uint32_t pairs = a.rot / 2, units = pairs + (a.dim - a.rot);
    const uint64_t th = id / units;
    const uint32_t u = (uint32_t)(id - th * units), token = (uint32_t)(th / a.heads), head = (uint32_t)(th - (uint64_t)token * a.heads);
    const T* x = (const T*)a.x + token * a.x_token + head * a.x_head;
    T* out = (T*)a.out + token * a.out_token + head * a.out_head;
    const uint64_t pos = a.positions ? (uint64_t)(int64_t)a.positions[token] : (uint64_t)a.first + token;
    uint32_t bad = 0;
    if (pos >= a.table_rows) bad = ZK_VALUES_POSITION;
    else if (u >= pairs) out[a.rot + (u - pairs)] = x[a.rot + (u - pairs)];
    else {
        const int2 cs = angle(a.table[pos * pairs + u], bad);
        const uint32_t i0 = a.neighbours ? 2 * u : u, i1 = a.neighbours ? 2 * u + 1 : u + pairs;
        const int64_t x0 = rope_get(x + i0, bad), x1 = rope_get(x + i1, bad);
        rope_put(out + i0, quotient<POW2>((int64_t)cs.x * (int32_t)x0 - (int64_t)cs.y * (int32_t)x1, a.sf), bad);
        rope_put(out + i1, quotient<POW2>((int64_t)cs.y * (int32_t)x0 + (int64_t)cs.x * (int32_t)x1, a.sf), bad);
    }
    raise(a.flag, bad);
}

// ---- products with a kept weight -----------------------------------------------------------------------------------------------------------------
// x and W as balanced base-256 digits (planes.hpp): an integer product is an int8 product for every pair of planes, pairs of equal weight 256^(i+j)
// in one int32 accumulator (at most three pairs of K 2^14, K below 2^17 / 3), the accumulators joined in 64 bits at the end.  Exact in any order.
struct Epilogue {
    int32_t* out;
    Divisor sf, sf_gate, sf_hidden;      // linear: sf; gated: sf is the up projection's
    const int32_t* table;
    int64_t low;
    uint32_t len;
    uint32_t* flag;
};
__device__ __forceinline__ int32_t gated_value(int64_t g, int64_t u, const Epilogue& e, uint32_t& bad) {
    const int64_t at = quotient_any(g, e.sf_gate) - e.low;
    if (at < 0 || at >= (int64_t)e.len) { bad |= ZK_VALUES_TABLE; return 0; }
    const int32_t up = narrow(quotient_any(u, e.sf), bad);
    return narrow(quotient_any((int64_t)e.table[at] * up, e.sf_hidden), bad);
}
// a weight's digit planes
struct Planes { const int8_t* p; uint32_t rows, Kp; int n; };
struct ProductArgs {
    const int32_t* x;
    size_t ldx;
    uint32_t rows, inner, cols;
    int x_aligned;                       // rows of x begin at multiples of 16 bytes
    Planes w, gate;                      // gated: w is the up projection
    const int8_t* px;                    // x's four planes, rows_padded rows each, and how many of them 32 rows' stretch of CHUNK columns needs
    const uint32_t* need;
    const int8_t* zeros;                 // 1 KB
    uint32_t rows_padded, chunks;
    Epilogue e;
};
static constexpr uint32_t CHUNK = 256;
// sum_s a[s] 256^s: below 2^62 in magnitude, or flagged and 0.  |a[s]| < 2^31, so the two low terms are below 2^41 together and the rest, in
// units of 2^16, says whether the sum fits 64 bits.
template <int NS> __device__ __forceinline__ int64_t joined(const int32_t (&a)[NS], uint32_t& bad) {
    int64_t lo = a[0], hi = 0;
    if constexpr (NS > 1) lo += (int64_t)a[1] << 8;
#pragma unroll
    for (int s = 2; s < NS; ++s) hi += (int64_t)a[s] << (8 * (s - 2));
    const int64_t limit = (1ll << 46) + (1ll << 25), most = 1ll << 62;
    if (hi >= limit || hi <= -limit) { bad |= ZK_VALUES_RANGE; return 0; }
    const int64_t v = hi * 65536 + lo;
    if (v >= most || v <= -most) { bad |= ZK_VALUES_RANGE; return 0; }
    return v;
}
// the digits of 16 values, plane by plane: plane j's 16 bytes in out[j]
__device__ __forceinline__ void digit_planes(const int32_t (&x)[16], v4i (&out)[4], uint32_t& bad) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bad |= x[4 * w + e] > 0x7F7F7F7F ? (uint32_t)ZK_VALUES_RANGE : 0u;      // four digits reach no further
            d[e] = digit_bytes((uint32_t)x[4 * w + e]);
        }
        const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), b = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
        const uint32_t c = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), e = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
        out[0][w] = (int)__builtin_amdgcn_perm(c, a, 0x05040100u);
        out[1][w] = (int)__builtin_amdgcn_perm(c, a, 0x07060302u);
        out[2][w] = (int)__builtin_amdgcn_perm(e, b, 0x05040100u);
        out[3][w] = (int)__builtin_amdgcn_perm(e, b, 0x07060302u);
    }
}
// 16 values of a row from column k on; zeros beyond the row's end and for rows that are none
__device__ __forceinline__ void row_piece(const ProductArgs& g, uint32_t row, uint32_t k, int32_t (&x)[16]) {
    const int32_t* p = g.x + row * g.ldx + k;
    if (row < g.rows && g.x_aligned && k + 16 <= g.inner) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const v4i v = reinterpret_cast<const v4i*>(p)[w];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * w + e] = v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = (row < g.rows && k + e < g.inner) ? p[e] : 0;
    }
}

// x's planes for the products of many rows.  A wave takes 32 rows and CHUNK columns, 32 columns at a time: a lane 16 values of a row, so that the wave
// writes 1 KB of every plane in one piece.  It notes how many planes its stretch needs, in a place of its own.
__global__ void __launch_bounds__(256) k_split_x(const ProductArgs g, int8_t* __restrict__ planes, uint32_t* __restrict__ need, v4i* __restrict__ zeros) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 64) zeros[threadIdx.x] = v4i{0, 0, 0, 0};
    const uint32_t lane = threadIdx.x & 63u, chunk = blockIdx.x * 4 + (threadIdx.x >> 6), group = blockIdx.y;
    if (chunk >= g.chunks) return;
    const uint32_t row = group * 32 + (lane >> 1), h = lane & 1u, Kp = g.w.Kp;
    uint32_t bad = 0, planes_needed = 1;
    for (uint32_t k0 = chunk * CHUNK; k0 < min((chunk + 1) * CHUNK, Kp); k0 += 32) {
        int32_t x[16];
        v4i d[4];
        row_piece(g, row, k0 + 16 * h, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t m = (uint32_t)(x[e] < 0 ? ~x[e] : x[e]);      // p digits hold -128 (256^p - 1) / 255 .. 127 (256^p - 1) / 255
            planes_needed = max(planes_needed, m <= 127u ? 1u : m <= 32639u ? 2u : m <= 8355711u ? 3u : 4u);
        }
        digit_planes(x, d, bad);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<v4i*>(planes + (size_t)j * g.rows_padded * Kp + plane_at(g.rows_padded, row, k0 + 16 * h)) = d[j];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) planes_needed = max(planes_needed, (uint32_t)__shfl_xor(planes_needed, off, 64));
    if (lane == 0) need[(size_t)group * g.chunks + chunk] = planes_needed;
    raise(g.e.flag, bad);
}

// Many rows.  A workgroup of four waves takes 64 MT rows by 128 columns of weights -- 64 of each where there are two: a wave's gate and up tiles lie in the same
// lanes, and what joins them needs no exchange -- and a wave 32 MT by 64, as 32 x 32 tiles of v_mfma_i32_32x32x32_i8.
// Steps of 32 contraction bytes go from memory to LDS without passing through registers, four buffers deep; a step's fragments are read while the step before
// is multiplied, since one wave a SIMD (256 accumulators with MT = 2) has nobody to cover for it.
template <bool GATED, int PA, int PB, int MT> struct Tile {
    static constexpr int NS = PA + PB - 1, TM = 64 * MT, PIECES = PA * 2 * MT + PB * 4, SHARE = (PIECES + 3) / 4, BYTES = (PA * TM + PB * 128) * 32;
    v16i acc[NS][MT][2];
    __device__ __forceinline__ void multiply(const ProductArgs& g, uint32_t m0, uint32_t n0, int8_t* const (&buf)[4]) {
        const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), wm = wave >> 1, wn = wave & 1;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[s][m][q][r] = 0;
        // The wave's pieces of a step: 32 rows of a plane each, x's first.  A weight's rows beyond the last read the last, a plane that it has not reads zeros.
        const int8_t* src[SHARE];              // the same for all lanes, as is the step
        uint32_t at[SHARE], dst[SHARE];
        size_t step[SHARE];
        const uint32_t lr = lane >> 1, lane_half = gemm_half(lr, lane & 1u) * 16;      // every piece begins at a multiple of 32 rows
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            const uint32_t c = min(wave + 4 * i, (uint32_t)PIECES - 1);
            if (c < PA * 2 * MT) {
                const uint32_t plane = c / (2 * MT), r = c % (2 * MT) * 32;
                src[i] = g.px + (size_t)plane * g.rows_padded * g.w.Kp + (size_t)(m0 + r) * 32;
                at[i] = lr * 32 + lane_half;
                dst[i] = (plane * TM + r) * 32;
                step[i] = (size_t)g.rows_padded * 32;
            } else {
                const uint32_t cb = c - PA * 2 * MT, plane = cb >> 2, r = (cb & 3u) * 32, first = n0 + (GATED ? r & 63u : r);
                const Planes& w = GATED && r < 64 ? g.gate : g.w;
                const bool has = (int)plane < w.n, inside = first < w.rows;
                src[i] = has ? w.p + (size_t)plane * w.rows * w.Kp + (size_t)(inside ? first : w.rows - 1) * 32 : g.zeros;
                at[i] = (has && inside ? min(lr, w.rows - 1 - first) : 0u) * 32 + lane_half;
                dst[i] = (PA * TM + plane * 128 + r) * 32;
                step[i] = has ? (size_t)w.rows * 32 : 0;
            }
        }
        const uint32_t half = lane >> 5, steps = g.w.Kp / 32;
        const uint32_t rowA = wm * 32 * MT + (lane & 31), at_a = rowA * 32 + gemm_half(rowA, half) * 16;
        const uint32_t rowB = wn * (GATED ? 32 : 64) + (lane & 31), next_b = GATED ? 64 : 32, at_b = (PA * TM + rowB) * 32 + gemm_half(rowB, half) * 16;      // 32 rows on: the same halves
        auto fetch = [&](int8_t* to) {                         // the next step
#pragma unroll
            for (int i = 0; i < SHARE; ++i) { load_to_lds(src[i] + at[i], to + dst[i]); src[i] += step[i]; }
        };
        struct Fragments { v4i a[PA][MT], b[PB][2]; };
        auto read = [&](const int8_t* from, Fragments& f) {
#pragma unroll
            for (int i = 0; i < PA; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m) f.a[i][m] = *reinterpret_cast<const v4i*>(from + at_a + (i * TM + 32 * m) * 32);
#pragma unroll
            for (int j = 0; j < PB; ++j)
#pragma unroll
                for (int q = 0; q < 2; ++q) f.b[j][q] = *reinterpret_cast<const v4i*>(from + at_b + (j * 128 + next_b * q) * 32);
        };
        auto products = [&](const Fragments& f) {
#pragma unroll
            for (int i = 0; i < PA; ++i)
#pragma unroll
                for (int j = 0; j < PB; ++j)
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int q = 0; q < 2; ++q) acc[i + j][m][q] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[i][m], f.b[j][q], acc[i + j][m][q], 0, 0, 0);
        };
        // the fragments' reads and the next loads spread over the products
        auto spread = [&](bool fetches) {
            constexpr int READS = PA * MT + PB * 2, PRODUCTS = PA * PB * MT * 2;
            static_assert(PRODUCTS >= READS + SHARE, "a product for every read and load");
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // an LDS read
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);      // a matrix instruction
            }
            if (fetches) {
#pragma unroll
                for (int i = 0; i < SHARE; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a load
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
            }
            __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
        };
        // Everybody's share of a step is in LDS when no more than `younger` steps' loads of a wave's own are on their way and all waves are past the barrier; with no LDS
        // read on its way either (lgkmcnt 0), the buffer read last is free for the next fetch.
        auto arrived = [&](auto younger) {
            constexpr int N = decltype(younger)::value * SHARE;
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        const std::integral_constant<int, 0> none;
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        const std::integral_constant<int, 3> three;
        Fragments even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) fetch(buf[i]);
        arrived(three);
        read(buf[0], even);
        for (uint32_t t = 4; t < steps; t += 4) {              // Kp is a multiple of 128: four steps or more
            arrived(two); fetch(buf[0]); read(buf[1], odd); products(even); spread(true);
            arrived(two); fetch(buf[1]); read(buf[2], even); products(odd); spread(true);
            arrived(two); fetch(buf[2]); read(buf[3], odd); products(even); spread(true);
            arrived(two); fetch(buf[3]); read(buf[0], even); products(odd); spread(true);
        }
        arrived(two); read(buf[1], odd); products(even); spread(false);
        arrived(one); read(buf[2], even); products(odd); spread(false);
        arrived(none); read(buf[3], odd); products(even); spread(false);
        products(odd);
        __syncthreads();                                       // a next tile's loads find buffers that nobody reads any more
    }
    __device__ __forceinline__ void finish(const ProductArgs& g, uint32_t m0, uint32_t n0, uint32_t& bad) {
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t row = m0 + (wm * MT + m) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                int64_t v[2];
                uint32_t off = 0;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    int32_t a[NS];
#pragma unroll
                    for (int s = 0; s < NS; ++s) a[s] = acc[s][m][q][r];
                    v[q] = joined<NS>(a, off);
                }
                if constexpr (GATED) {
                    const uint32_t col = n0 + wn * 32 + (lane & 31);
                    if (row < g.rows && col < g.cols) {
                        g.e.out[(size_t)row * g.cols + col] = gated_value(v[0], v[1], g.e, off);
                        bad |= off;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t col = n0 + wn * 64 + q * 32 + (lane & 31);
                        if (row < g.rows && col < g.cols) {
                            uint32_t one = 0;
                            g.e.out[(size_t)row * g.cols + col] = narrow(quotient_any(v[q], g.e.sf), one);
                            bad |= one | off;
                        }
                    }
                }
            }
    }
};
template <bool GATED, int PB, int MT> __global__ void __launch_bounds__(256, MT == 2 || PB == 3 ? 1 : 2) k_product(const ProductArgs g) {
    constexpr int BYTES = Tile<GATED, 3, PB, MT>::BYTES > Tile<GATED, 4, PB, 1>::BYTES ? Tile<GATED, 3, PB, MT>::BYTES : Tile<GATED, 4, PB, 1>::BYTES;
    // a variable a buffer: the compiler waits for a direct load before every read of the variable that it writes
    __shared__ __attribute__((aligned(16))) int8_t s0[BYTES], s1[BYTES], s2[BYTES], s3[BYTES];
    // Workgroups go to the eight dies in turn: a die takes a run of tiles in groups of eight rows of them, which share operands in its L2
    uint32_t tm = blockIdx.y, tn = blockIdx.x;
    {
        const uint32_t nx = gridDim.x, ny = gridDim.y, total = nx * ny, id = blockIdx.y * nx + blockIdx.x;
        if ((total & 7u) == 0 && total >= 64) {
            const uint32_t lin = (id & 7u) * (total >> 3) + (id >> 3), group = lin / (8 * nx), first = group * 8, rows = ny - first < 8 ? ny - first : 8u, in = lin - group * 8 * nx;
            tm = first + in % rows;
            tn = in / rows;
        }
    }
    const uint32_t m0 = tm * 64 * MT, n0 = tn * (GATED ? 64 : 128);
    uint32_t need = 0, bad = 0;
    for (uint32_t i = threadIdx.x & 63u; i < 2 * MT * g.chunks; i += 64) need = max(need, g.need[(size_t)(m0 / 32) * g.chunks + i]);
    const bool wide = __any(need > 3);
    int8_t* const buf[4] = {s0, s1, s2, s3};
    if (!wide) {
        Tile<GATED, 3, PB, MT> t;
        t.multiply(g, m0, n0, buf);
        t.finish(g, m0, n0, bad);
    } else {                                   // a value of more than three digits: all four planes, 64 rows at a time
        for (uint32_t m = m0; m < m0 + 64 * MT; m += 64) {
            Tile<GATED, 4, PB, 1> t;
            t.multiply(g, m, n0, buf);
            t.finish(g, m, n0, bad);
        }
    }
    raise(g.e.flag, bad);
}

// Few rows: the weights are read once and nothing else counts.  A workgroup takes 16 columns (of each weight), its waves the units of 64 contraction bytes in
// turn, straight from memory into the fragments of v_mfma_i32_16x16x64_i8 -- a fragment of 16 columns is two pieces of 512 bytes in the planes' layout.  x is
// split on the way, all four digits (the matrix cores idle anyway).  The waves' accumulators are added up in LDS, integers in any order.
template <bool GATED, int PB, int RT> __global__ void __launch_bounds__(512) k_product_few(const ProductArgs g) {
    constexpr int MATS = GATED ? 2 : 1, NS = 4 + PB - 1, WAVES = 8, DEPTH = RT == 1 ? 4 : 2;
    __shared__ int32_t sum[NS * MATS * RT][256];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = lane & 15u, q = lane >> 4;
    const uint32_t units = g.w.Kp / 64, col = min(blockIdx.x * 16 + c, g.cols - 1);
    for (uint32_t i = threadIdx.x; i < NS * MATS * RT * 256; i += 512) (&sum[0][0])[i] = 0;
    const int8_t* src[MATS][PB];
    const Planes* mats[2] = {GATED ? &g.gate : &g.w, &g.w};
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int j = 0; j < PB; ++j)
            src[m][j] = mats[m]->p + (size_t)(j < mats[m]->n ? j : 0) * mats[m]->rows * g.w.Kp + ((size_t)(q >> 1) * g.cols + col) * 32 + (q & 1u) * 16;
    v4i acc[NS][MATS][RT];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[s][m][r] = v4i{0, 0, 0, 0};
    v4i w[DEPTH][MATS][PB];
    int32_t x[DEPTH][RT][16];
    uint32_t bad = 0;
    auto load = [&](uint32_t u, int d) {
        u = min(u, units - 1);                 // behind the last one that again: never multiplied
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int j = 0; j < PB; ++j) w[d][m][j] = *reinterpret_cast<const v4i*>(src[m][j] + (size_t)u * 2 * g.cols * 32);
#pragma unroll
        for (int r = 0; r < RT; ++r) row_piece(g, r * 16 + c, u * 64 + q * 16, x[d][r]);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(wave + d * WAVES, d);
    for (uint32_t u0 = wave; u0 < units; u0 += DEPTH * WAVES)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const uint32_t u = u0 + d * WAVES;
            if (u < units) {
                const v4i zero = {0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < MATS; ++m)
#pragma unroll
                    for (int j = 1; j < PB; ++j)
                        if (j >= mats[m]->n) w[d][m][j] = zero;
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    v4i a[4];
                    digit_planes(x[d][r], a, bad);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < PB; ++j)
#pragma unroll
                            for (int m = 0; m < MATS; ++m) acc[i + j][m][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], w[d][m][j], acc[i + j][m][r], 0, 0, 0);
                }
            }
            load(u + DEPTH * WAVES, d);
        }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) atomicAdd(&sum[(s * MATS + m) * RT + r][(4 * q + e) * 16 + c], acc[s][m][r][e]);      // row 4 q + e, column c
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < RT * 256; i += 512) {
        const uint32_t r = i >> 8, row = i >> 4, out_col = blockIdx.x * 16 + (i & 15u);
        if (row >= g.rows || out_col >= g.cols) continue;
        int64_t v[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            int32_t a[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) a[s] = sum[(s * MATS + m) * RT + r][i & 255u];
            v[m] = joined<NS>(a, bad);
        }
        int32_t y;
        if constexpr (GATED) y = gated_value(v[0], v[1], g.e, bad);
        else y = narrow(quotient_any(v[0], g.e.sf), bad);
        g.e.out[(size_t)row * g.cols + out_col] = y;
    }
    raise(g.e.flag, bad);
}

// ---- a weight's planes from its int32 form ---------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_absmax_i32(unsigned long long* __restrict__ out, const int32_t* __restrict__ a, size_t n) {
    uint32_t m = 0;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const int64_t v = a[i];
        const uint32_t mag = (uint32_t)(v < 0 ? -v : v);
        m = mag > m ? mag : m;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { const uint32_t o = __shfl_xor(m, off, 64); m = o > m ? o : m; }
    if ((threadIdx.x & 63u) == 0 && m) atomicMax(out, (unsigned long long)m);
}
// grid (P tiles of 64, K tiles of 64): a 64 x 64 tile goes through LDS so that reads run along p and writes along k
__global__ void __launch_bounds__(256) k_split_cols_i32(int8_t* __restrict__ planes, const int32_t* __restrict__ B, uint32_t N, uint32_t P, uint32_t Kp, int np) {
    __shared__ __attribute__((aligned(16))) int8_t tile[4][64][80];
    const uint32_t t = threadIdx.x, p = t & 63, kq = t >> 6, p0 = blockIdx.x * 64, k0 = blockIdx.y * 64;
    for (int r = 0; r < 16; ++r) {
        const uint32_t k = k0 + kq * 16 + r;
        const uint32_t d = digit_bytes((k < N && p0 + p < P) ? (uint32_t)B[(size_t)k * P + p0 + p] : 0u);
        for (int j = 0; j < 4; ++j) tile[j][p][kq * 16 + r] = (int8_t)(d >> (8 * j));
    }
    __syncthreads();
    const uint32_t row = t >> 2, ch = t & 3;
    if (p0 + row < P)
        for (int j = 0; j < np; ++j)
            *reinterpret_cast<v4i*>(planes + (size_t)j * P * Kp + plane_at(P, p0 + row, k0 + ch * 16)) = *reinterpret_cast<const v4i*>(&tile[j][row][ch * 16]);
}

// ---- entry points -----------------------------------------------------------------------------------------------------------------------------------
// The flag of a call: the caller's, or one of the call's own that is looked at before the call returns.
struct CallFlag {
    uint32_t* dev = nullptr;
    std::unique_ptr<Scratch> own;
    hipStream_t st;
    int begin(void* flag_dev, hipStream_t stream, const char* name) {
        st = stream;
        dev = (uint32_t*)flag_dev;
        if (dev) return 0;
        if (const int rc = not_captured(stream, name)) return rc;
        own.reset(new Scratch(4, stream));
        if (own->rc) return own->rc;
        dev = own->as<uint32_t>();
        return clear_words(dev, 1, stream);
    }
    // what a call without a flag of the caller's, or without a workspace, does cannot be captured: it waits, and its memory goes back to the pool
    static int not_captured(hipStream_t stream, const char* name) {
        if (!stream) return 0;
        hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
        ZK_HIP(hipStreamIsCapturing(stream, &s));
        if (s != hipStreamCaptureStatusNone) {
            set_error(ZK_ERR_ARG, std::string(name) + ": a captured call needs a flag and a workspace of the caller's");
            return ZK_ERR_ARG;
        }
        return 0;
    }
    int end(const char* name) {
        if (!own) return 0;
        void* stage = nullptr;
        if (const int rc = staging(&stage, 4)) return rc;
        ZK_HIP(hipMemcpyAsync(stage, dev, 4, hipMemcpyDeviceToHost, st));
        ZK_HIP(hipStreamSynchronize(st));
        uint32_t bad = 0;
        memcpy(&bad, stage, 4);
        if (!bad) return 0;
        const char* what = (bad & ZK_VALUES_TABLE) ? ": an activation lies outside the table" : (bad & ZK_VALUES_POSITION) ? ": a position lies outside the table" : ": a value does not fit";
        set_error(ZK_ERR_ARG, std::string(name) + what);
        return ZK_ERR_ARG;
    }
};

static constexpr uint32_t MAX_INNER = (1u << 17) / 3;      // three plane pairs of 2^14 a term in an int32 accumulator
static int check_weight(const MatmulRhs* w, const char* name) {
    ZK_ARG(w != nullptr, std::string(name) + ": null weight");
    ZK_ARG(w->planes != nullptr && w->pb >= 1 && w->pb <= 3, std::string(name) + ": the weight has elements beyond 8355711 (three digits of eight bits)");
    ZK_ARG(w->N <= MAX_INNER, std::string(name) + ": an inner dimension above 43690");
    return 0;
}
static Planes planes_of(const MatmulRhs* w) { return Planes{(const int8_t*)w->planes, w->P, w->Kp, w->pb}; }

static constexpr uint32_t FEW_ROWS = 32;
static size_t padded_rows(uint32_t rows) { return ((size_t)rows + 127) / 128 * 128; }
template <bool GATED, int PB> static void launch_few(const ProductArgs& g, hipStream_t st) {
    if (g.rows <= 16) hipLaunchKernelGGL((k_product_few<GATED, PB, 1>), dim3(cdiv(g.cols, 16)), dim3(512), 0, st, g);
    else hipLaunchKernelGGL((k_product_few<GATED, PB, 2>), dim3(cdiv(g.cols, 16)), dim3(512), 0, st, g);
}
template <bool GATED, int PB> static void launch_many(const ProductArgs& g, hipStream_t st) {
    const unsigned tn = cdiv(g.cols, GATED ? 64 : 128);
    if constexpr (PB == 2) if ((size_t)tn * cdiv(g.rows, 128) >= 256) {
        hipLaunchKernelGGL((k_product<GATED, PB, 2>), dim3(tn, cdiv(g.rows, 128)), dim3(256), 0, st, g);
        return;
    }
    hipLaunchKernelGGL((k_product<GATED, PB, 1>), dim3(tn, cdiv(g.rows, 64)), dim3(256), 0, st, g);
}
template <bool GATED> static int product(const char* name, ProductArgs& g, void* flag_dev, void* workspace, size_t workspace_bytes, hipStream_t st) {
    ZK_ARG(g.x != nullptr && g.e.out != nullptr, std::string(name) + ": null tensor");
    ZK_ARG(g.ldx >= g.inner, std::string(name) + ": rows of x overlap (ldx below the inner dimension)");
    ZK_ARG(g.rows <= (1u << 18), std::string(name) + ": more than 262144 rows in one call");
    ZK_ARG(workspace == nullptr || workspace_bytes >= zk_i32_linear_workspace(g.rows, g.inner), std::string(name) + ": the workspace is smaller than zk_i32_linear_workspace says");
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    g.e.flag = flag.dev;
    g.x_aligned = (g.ldx & 3) == 0 && ((uintptr_t)g.x & 15) == 0;
    const int pb = std::max(g.w.n, GATED ? g.gate.n : 0);
    if (g.rows <= FEW_ROWS) {
        if (pb <= 2) launch_few<GATED, 2>(g, st);
        else launch_few<GATED, 3>(g, st);
        ZK_LAUNCH_CHECK();
        return flag.end(name);
    }
    const size_t bytes = zk_i32_linear_workspace(g.rows, g.inner);
    std::unique_ptr<Scratch> own;
    if (!workspace) {
        if (const int rc = CallFlag::not_captured(st, name)) return rc;
        own.reset(new Scratch(bytes, st));
        if (own->rc) return own->rc;
        workspace = own->p;
    }
    ZK_ARG(((uintptr_t)workspace & 15) == 0, std::string(name) + ": the workspace must begin at a multiple of 16 bytes");
    g.rows_padded = padded_rows(g.rows);
    g.chunks = cdiv(g.w.Kp, CHUNK);
    g.px = (const int8_t*)workspace;
    g.zeros = g.px + (size_t)4 * g.rows_padded * g.w.Kp;
    g.need = (const uint32_t*)(g.zeros + 1024);
    hipLaunchKernelGGL(k_split_x, dim3(cdiv(g.chunks, 4), g.rows_padded / 32), dim3(256), 0, st, g, (int8_t*)workspace, (uint32_t*)g.need, (v4i*)g.zeros);
    if (pb <= 2) launch_many<GATED, 2>(g, st);
    else launch_many<GATED, 3>(g, st);
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}

extern "C" {

int zk_i32_residual_norm(void* h, void* n, void* rms_inv, const void* x, size_t ldx, const void* b, size_t ldb, const void* post, const void* gate, uint32_t gate_rows, int32_t res,
                         const void* w, uint32_t rows, uint32_t cols, double eps, double scale, uint32_t sf, void* flag_dev, void* stv) {
    if (rows == 0) return 0;
    ZK_ARG(x != nullptr && cols > 0 && (h != nullptr || n != nullptr || rms_inv != nullptr), "zk_i32_residual_norm: null x, no output or empty rows");
    ZK_ARG(n == nullptr || w != nullptr, "zk_i32_residual_norm: a normed output needs a weight");
    ZK_ARG(ldx >= cols && (b == nullptr || ldb >= cols), "zk_i32_residual_norm: rows overlap (leading dimension below cols)");
    ZK_ARG(b != nullptr || (post == nullptr && gate == nullptr), "zk_i32_residual_norm: a norm behind the block or a gate needs the block's output");
    ZK_ARG((gate == nullptr) == (gate_rows == 0) && (gate == nullptr || rows % gate_rows == 0), "zk_i32_residual_norm: gate_rows must divide rows, and be 0 without a gate");
    ZK_ARG(sf > 0, "zk_i32_residual_norm: a scaling factor of 0");
    ZK_ARG(scale > 0 && eps > 0 && scale <= 1e18 && scale >= 1e-18 && scale / std::sqrt(eps) <= 2147483000.0, "zk_i32_residual_norm: scale and eps must be positive, scale / sqrt(eps) below 2^31");
    ZK_ARG(rows <= 0x7FFFFFFFu, "zk_i32_residual_norm: too many rows in one call");
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, "zk_i32_residual_norm")) return rc;
    int e2 = 0;
    const NormArgs a{(int32_t*)h, (int32_t*)n, (int32_t*)rms_inv, (const int32_t*)x, (const int32_t*)b, (const int32_t*)post, (const int32_t*)gate, (const int32_t*)w, ldx, ldb, cols,
                     gate ? rows / gate_rows : 1, res, scale, eps, std::frexp(scale, &e2) == 0.5, divisor(sf), flag.dev};
    if (a.sf.shift >= 0) hipLaunchKernelGGL(k_residual_norm_long<true>, dim3(rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_residual_norm_long<false>, dim3(rows), dim3(256), 0, st, a);
    ZK_LAUNCH_CHECK();
    return flag.end("zk_i32_residual_norm");
}

static int rope(const char* name, bool fr, void* out, size_t out_token, size_t out_head, const void* x, size_t x_token, size_t x_head, uint32_t tokens, uint32_t heads, uint32_t dim, uint32_t rot,
                int neighbours, const void* table, uint32_t table_rows, const void* positions, uint32_t first, uint32_t sf, void* flag_dev, void* stv) {
    if (tokens == 0 || heads == 0) return 0;
    ZK_ARG(out != nullptr && x != nullptr && dim > 0, std::string(name) + ": null tensor or empty heads");
    ZK_ARG(rot <= dim && rot % 2 == 0, std::string(name) + ": the rotated part must be even and within the head");
    ZK_ARG(rot == 0 || (table != nullptr && table_rows > 0), std::string(name) + ": no table");
    ZK_ARG(sf > 0 && sf <= (1u << 30), std::string(name) + ": the table's scale must be 1 .. 2^30");
    ZK_ARG(out != x || (out_token == x_token && out_head == x_head), std::string(name) + ": in place with other strides");
    ZK_ARG((tokens == 1 || (x_token >= dim && out_token >= dim)) && (heads == 1 || (x_head >= dim && out_head >= dim)), std::string(name) + ": heads overlap (a stride below the head's width)");
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    const RopeArgs a{out, x, out_token, out_head, x_token, x_head, tokens, heads, dim, rot, neighbours, (const int2*)table, rot ? table_rows : 0xFFFFFFFFu, (const int32_t*)positions, first, divisor(sf), flag.dev};
    const uint64_t total = (uint64_t)tokens * heads * (rot / 2 + (dim - rot)), step = 1ull << 30;
    for (uint64_t base = 0; base < total; base += step) {
        const uint64_t end = std::min(total, base + step);
        const dim3 grid(cdiv(end - base, 256));
        if (fr) {
            if (a.sf.shift >= 0) hipLaunchKernelGGL((k_rope<Fr, true>), grid, dim3(256), 0, st, a, base, end);
            else hipLaunchKernelGGL((k_rope<Fr, false>), grid, dim3(256), 0, st, a, base, end);
        } else {
            if (a.sf.shift >= 0) hipLaunchKernelGGL((k_rope<int32_t, true>), grid, dim3(256), 0, st, a, base, end);
            else hipLaunchKernelGGL((k_rope<int32_t, false>), grid, dim3(256), 0, st, a, base, end);
        }
    }
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}
int zk_i32_rope(void* out, size_t out_token, size_t out_head, const void* x, size_t x_token, size_t x_head, uint32_t tokens, uint32_t heads, uint32_t dim, uint32_t rot, int neighbours,
                const void* table, uint32_t table_rows, const void* positions, uint32_t first, uint32_t sf, void* flag_dev, void* stv) {
    return rope("zk_i32_rope", false, out, out_token, out_head, x, x_token, x_head, tokens, heads, dim, rot, neighbours, table, table_rows, positions, first, sf, flag_dev, stv);
}
int zk_fr_rope(void* out, size_t out_token, size_t out_head, const void* x, size_t x_token, size_t x_head, uint32_t tokens, uint32_t heads, uint32_t dim, uint32_t rot, int neighbours,
               const void* table, uint32_t table_rows, const void* positions, uint32_t first, uint32_t sf, void* flag_dev, void* stv) {
    return rope("zk_fr_rope", true, out, out_token, out_head, x, x_token, x_head, tokens, heads, dim, rot, neighbours, table, table_rows, positions, first, sf, flag_dev, stv);
}

int zk_i32_rhs_prepare(void** prepared, const void* B, uint32_t N, uint32_t P, void* stv) {
    hipStream_t st = (hipStream_t)stv;
    ZK_ARG(prepared != nullptr && B != nullptr && N > 0 && P > 0, "zk_i32_rhs_prepare: null argument or empty matrix");
    ZK_ARG(N <= MAX_INNER && P <= (1u << 30), "zk_i32_rhs_prepare: an inner dimension above 43690, or too many columns");
    if (const int rc = CallFlag::not_captured(st, "zk_i32_rhs_prepare")) return rc;
    std::unique_ptr<MatmulRhs> r(new MatmulRhs);
    r->N = N; r->P = P; r->Kp = (N + GBK - 1) / GBK * GBK;
    {
        Scratch mx(8, st);
        if (mx.rc) return mx.rc;
        if (const int rc = clear_words(mx.p, 2, st)) return rc;
        const size_t nb = (size_t)N * P;
        hipLaunchKernelGGL(k_absmax_i32, dim3((unsigned)std::min<size_t>(2048, nb / 2048 + 1)), dim3(256), 0, st, mx.as<unsigned long long>(), (const int32_t*)B, nb);
        ZK_LAUNCH_CHECK();
        void* stage = nullptr;
        if (const int rc = staging(&stage, 8)) return rc;
        ZK_HIP(hipMemcpyAsync(stage, mx.p, 8, hipMemcpyDeviceToHost, st));
        ZK_HIP(hipStreamSynchronize(st));
        memcpy(&r->mb, stage, 8);
    }
    r->pb = digits_for(r->mb);
    ZK_ARG(r->pb >= 1 && r->pb <= 3, "zk_i32_rhs_prepare: the weight has elements beyond 8355711 (three digits of eight bits)");
    if (const int rc = pool_alloc(&r->planes, (size_t)r->pb * P * r->Kp, st)) return rc;
    hipLaunchKernelGGL(k_split_cols_i32, dim3(cdiv(P, 64), r->Kp / 64), dim3(256), 0, st, (int8_t*)r->planes, (const int32_t*)B, N, P, r->Kp, r->pb);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { (void)pool_free(r->planes, st); return hip_fail(e, "k_split_cols_i32", __FILE__, __LINE__); }
    *prepared = r.release();
    return 0;
}
size_t zk_i32_linear_workspace(uint32_t rows, uint32_t inner) {
    const size_t Kp = ((size_t)inner + GBK - 1) / GBK * GBK;
    if (rows <= FEW_ROWS) return 0;
    return padded_rows(rows) * Kp * 4 + 1024 + padded_rows(rows) / 32 * ((Kp + CHUNK - 1) / CHUNK) * 4;
}
int zk_i32_linear(void* out, const void* x, size_t ldx, const void* prepared, uint32_t rows, uint32_t sf, void* workspace, size_t workspace_bytes, void* flag_dev, void* stv) {
    const MatmulRhs* w = (const MatmulRhs*)prepared;
    if (const int rc = check_weight(w, "zk_i32_linear")) return rc;
    ZK_ARG(sf > 0, "zk_i32_linear: a scaling factor of 0");
    if (rows == 0) return 0;
    ProductArgs g{};
    g.x = (const int32_t*)x; g.ldx = ldx; g.rows = rows; g.inner = w->N; g.cols = w->P; g.w = planes_of(w);
    g.e.out = (int32_t*)out; g.e.sf = divisor(sf);
    return product<false>("zk_i32_linear", g, flag_dev, workspace, workspace_bytes, (hipStream_t)stv);
}
int zk_i32_gated(void* out, const void* x, size_t ldx, const void* gate_prepared, const void* up_prepared, uint32_t rows, uint32_t sf_gate, uint32_t sf_up, const void* table, int32_t low,
                 uint32_t len, uint32_t sf_hidden, void* workspace, size_t workspace_bytes, void* flag_dev, void* stv) {
    const MatmulRhs *w = (const MatmulRhs*)up_prepared, *gate = (const MatmulRhs*)gate_prepared;
    if (const int rc = check_weight(gate, "zk_i32_gated")) return rc;
    if (const int rc = check_weight(w, "zk_i32_gated")) return rc;
    ZK_ARG(w->N == gate->N && w->P == gate->P, "zk_i32_gated: the two projections have different shapes");
    ZK_ARG(sf_gate > 0 && sf_up > 0 && sf_hidden > 0, "zk_i32_gated: a scaling factor of 0");
    ZK_ARG(table != nullptr && len > 0, "zk_i32_gated: no table of function values");
    if (rows == 0) return 0;
    ProductArgs g{};
    g.x = (const int32_t*)x; g.ldx = ldx; g.rows = rows; g.inner = w->N; g.cols = w->P; g.w = planes_of(w); g.gate = planes_of(gate);
    g.e.out = (int32_t*)out; g.e.sf = divisor(sf_up); g.e.sf_gate = divisor(sf_gate); g.e.sf_hidden = divisor(sf_hidden);
    g.e.table = (const int32_t*)table; g.e.low = low; g.e.len = len;
    return product<true>("zk_i32_gated", g, flag_dev, workspace, workspace_bytes, (hipStream_t)stv);
}

}  // extern "C"
