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
#include "detmath.hpp"
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
__device__ __forceinline__ int32_t narrow(int64_t v, uint32_t& bad) {
    bad |= (int32_t)(v >> 32) != ((int32_t)v >> 31) ? (uint32_t)ZK_VALUES_RANGE : 0u;
    return (int32_t)v;
}
__device__ __forceinline__ void raise(uint32_t* flag, uint32_t bad) { if (bad) atomicOr(flag, bad); }

// ---- norms with the residual stream -------------------------------------------------------------------------------------------------------
struct NormArgs {
    int32_t *h, *n, *rms_inv;
    const int32_t *x, *b, *post, *gate, *w;
    size_t ldx, ldb, row0;    // row0: the launch's first row
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

// A workgroup a row, VEC neighbouring columns NV times in each lane's registers: every tensor is read once and written once, which is what
// bounds it (2048 x 4096, x and b to h and n, 134 MB: 24 us, 5.6 TB/s; a copy of a gigabyte reaches 5.15).  One row of 4096: 4.5 us, two reductions and the way to memory and back.
// Rows whose squares add up to more than 2^53 -- one value beyond 2^26.5, 1449 at scale 2^16, is enough -- are added up by one lane out of LDS, 8 ns a term: a row of 4096 takes 32 us
// more, 2048 x 4096 107 us where one row in 64 is such a row and 182 where all are.
template <int VEC> __device__ __forceinline__ void row_load(int32_t (&v)[VEC], const int32_t* p) {
    if constexpr (VEC == 4) {
        const v4i q = *reinterpret_cast<const v4i*>(p);
        v[0] = q[0]; v[1] = q[1]; v[2] = q[2]; v[3] = q[3];
    } else v[0] = *p;
}
// STREAM: stores go past the caches, in the kernel for 512 rows and more of 1025 to 4096 columns (2048 x 4096: 31 us, 23 so, 512 x 4096 9.0 and 8.0, 8192 x 4096 104 and 102; with the projection
// that reads them behind it 206 either way); the other kernels' do not.
template <int VEC, bool STREAM> __device__ __forceinline__ void row_store(int32_t* p, const int32_t (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const v4i q = {v[0], v[1], v[2], v[3]};
        if constexpr (STREAM) __builtin_nontemporal_store(q, reinterpret_cast<v4i*>(p));
        else *reinterpret_cast<v4i*>(p) = q;
    } else *p = v[0];
}
template <int NV, int VEC, bool POW2, int THREADS> __global__ void __launch_bounds__(THREADS) k_residual_norm(const NormArgs a) {
    extern __shared__ double term[];           // blockDim.x * VEC
    __shared__ unsigned long long red_s[16];
    __shared__ uint32_t red_m[16];
    __shared__ double total;
    const size_t row = a.row0 + blockIdx.x;
    const uint32_t stride = blockDim.x * VEC, first = threadIdx.x * VEC;
    uint32_t bad = 0;
    auto load = [&](int32_t (&v)[NV][VEC], const int32_t* p) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (first + i * stride < a.cols) row_load<VEC>(v[i], p + first + i * stride);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = 0;
        }
    };
    auto store = [&](int32_t* p, const int32_t (&v)[NV][VEC]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) if (first + i * stride < a.cols) row_store<VEC, THREADS == 512>(p + first + i * stride, v[i]);
    };
    auto statistic = [&](const int32_t (&v)[NV][VEC]) {
        unsigned long long s = 0;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int32_t x = v[i][e];
                s += (unsigned long long)((int64_t)x * x);
                m = max(m, x < 0 ? 0u - (uint32_t)x : (uint32_t)x);
            }
        block_sum_max(s, m, red_s, red_m);
        if (sum_is_exact(s, m, a)) return rms_inverse((double)s / a.scale / a.scale, a);
        double acc = 0.0;                      // in index order, a stretch of `stride` terms at a time
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const double x = (double)v[i][e] / a.scale;
                term[first + e] = x * x;
            }
            __syncthreads();
            if (threadIdx.x == 0 && i * stride < a.cols) {
                const uint32_t cnt = min(a.cols - i * stride, stride);
                for (uint32_t q = 0; q < cnt; ++q) acc += term[q];
            }
        }
        if (threadIdx.x == 0) total = acc;
        __syncthreads();
        const double t = total;
        __syncthreads();
        return rms_inverse(t, a);
    };
    int32_t v[NV][VEC], w[NV][VEC];
    load(v, a.x + row * a.ldx);
    if (a.b) {
        int32_t q[NV][VEC], post[NV][VEC], gate[NV][VEC];
        load(q, a.b + row * a.ldb);
        if (a.post) load(post, a.post);
        if (a.gate) load(gate, a.gate + row / a.rows_per_gate * a.cols);
        if (a.n) load(w, a.w);
        if (a.post) {
            const int32_t r = statistic(q);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) q[i][e] = normed<POW2>(post[i][e], r, q[i][e], a.sf, bad);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                int32_t y = q[i][e];
                if (a.gate) y = narrow(quotient<POW2>((int64_t)gate[i][e] * y, a.sf), bad);
                v[i][e] = narrow((int64_t)v[i][e] + quotient<POW2>((int64_t)a.res * y, a.sf), bad);
            }
    } else if (a.n) load(w, a.w);
    if (a.h) store(a.h + row * a.cols, v);
    if (a.n || a.rms_inv) {
        const int32_t r = statistic(v);
        if (a.rms_inv && threadIdx.x == 0) a.rms_inv[row] = r;
        if (a.n) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = normed<POW2>(w[i][e], r, v[i][e], a.sf, bad);
            store(a.n + row * a.cols, v);
        }
    }
    raise(a.flag, bad);
}
// Rows too long for that: every pass reads the row again.  A lane writes only columns that it alone reads, so h and n may be x or b themselves.
template <bool POW2> __global__ void __launch_bounds__(256) k_residual_norm_long(const NormArgs a) {
    __shared__ unsigned long long red_s[4];
    __shared__ uint32_t red_m[4];
    __shared__ double term[256], total;
    const size_t row = a.row0 + blockIdx.x;
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
    int64_t v;
    if (!fr_fits_i64(*p, v) || v != (int64_t)(int32_t)v) { bad |= ZK_VALUES_RANGE; return 0; }
    return v;
}
__device__ __forceinline__ void rope_put(int32_t* p, int64_t v, uint32_t& bad) { *p = narrow(v, bad); }
// an element in two stores of 16 bytes, one behind the other: left to itself the compiler joins this place with the one that only copies, and splits or parts
// the stores that they share (20 of 80 rotated: 136 us instead of 105)
__device__ __forceinline__ void store_element(Fr* p, const Fr& e) {
    v4i* q = reinterpret_cast<v4i*>(p);
    q[0] = v4i{(int)e.v[0], (int)e.v[1], (int)e.v[2], (int)e.v[3]};
    q[1] = v4i{(int)e.v[4], (int)e.v[5], (int)e.v[6], (int)e.v[7]};
}
__device__ __forceinline__ void rope_put(Fr* p, int64_t v, uint32_t&) { store_element(p, fr_from_i64(v)); }
__device__ __forceinline__ void rope_copy(int32_t* to, const int32_t* from, uint32_t&) { *to = *from; }
__device__ __forceinline__ void rope_copy(Fr* to, const Fr* from, uint32_t& bad) {
    Fr e = *from;
    int64_t v;
    if (!fr_fits_i64(e, v) || v != (int64_t)(int32_t)v) { bad |= ZK_VALUES_RANGE; e = big_zero<8>(); }
    store_element(to, e);
    asm volatile("" ::: "memory");
}
// A lane VEC pairs of the rotated part or VEC elements of the rest; the heads of a token read its angles from the caches.  HBM: 16384 tokens of 32 x 128 int32 92 us,
// 5.9 TB/s (a pair a lane 143; 51 heads of 80, 20 rotated, which take that, 274); 2048 tokens of field elements 101 us, 5.3 TB/s; the launches of a token's 64 heads 3 us.
template <typename T, int VEC, bool POW2> __global__ void __launch_bounds__(256) k_rope(const RopeArgs a, uint32_t token0, uint32_t total) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const uint32_t pairs = a.rot / 2, groups = pairs / VEC, units = groups + (a.dim - a.rot) / VEC;
    const uint32_t th = id / units, u = id - th * units, t = th / a.heads, head = th - t * a.heads;
    const size_t token = (size_t)token0 + t;
    const T* x = (const T*)a.x + token * a.x_token + head * a.x_head;
    T* out = (T*)a.out + token * a.out_token + head * a.out_head;
    const uint64_t pos = a.positions ? (uint64_t)(int64_t)a.positions[token] : (uint64_t)a.first + token;
    uint32_t bad = 0;
    if (pos >= a.table_rows) bad = ZK_VALUES_POSITION;
    else if (u >= groups) {
        const uint32_t i = a.rot + (u - groups) * VEC;
        if constexpr (VEC == 4) *reinterpret_cast<v4i*>(out + i) = *reinterpret_cast<const v4i*>(x + i);
        else rope_copy(out + i, x + i, bad);
    } else if constexpr (VEC == 4) {
        const int2* cs = a.table + pos * pairs + 4 * u;
        const v4i c0 = *reinterpret_cast<const v4i*>(cs), c1 = *reinterpret_cast<const v4i*>(cs + 2);
        const uint32_t i0 = a.neighbours ? 8 * u : 4 * u, i1 = a.neighbours ? 8 * u + 4 : 4 * u + pairs;
        const v4i p = *reinterpret_cast<const v4i*>(x + i0), q = *reinterpret_cast<const v4i*>(x + i1);
        const int32_t x0[4] = {p[0], a.neighbours ? p[2] : p[1], a.neighbours ? q[0] : p[2], a.neighbours ? q[2] : p[3]};
        const int32_t x1[4] = {a.neighbours ? p[1] : q[0], a.neighbours ? p[3] : q[1], a.neighbours ? q[1] : q[2], q[3]};
        int32_t y0[4], y1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int2 k = angle(make_int2(e < 2 ? c0[2 * e] : c1[2 * e - 4], e < 2 ? c0[2 * e + 1] : c1[2 * e - 3]), bad);
            y0[e] = narrow(quotient<POW2>((int64_t)k.x * x0[e] - (int64_t)k.y * x1[e], a.sf), bad);
            y1[e] = narrow(quotient<POW2>((int64_t)k.y * x0[e] + (int64_t)k.x * x1[e], a.sf), bad);
        }
        *reinterpret_cast<v4i*>(out + i0) = a.neighbours ? v4i{y0[0], y1[0], y0[1], y1[1]} : v4i{y0[0], y0[1], y0[2], y0[3]};
        *reinterpret_cast<v4i*>(out + i1) = a.neighbours ? v4i{y0[2], y1[2], y0[3], y1[3]} : v4i{y1[0], y1[1], y1[2], y1[3]};
    } else {
        const int2 cs = angle(a.table[pos * pairs + u], bad);
        const uint32_t i0 = a.neighbours ? 2 * u : u, i1 = a.neighbours ? 2 * u + 1 : u + pairs;
        const int64_t x0 = rope_get(x + i0, bad), x1 = rope_get(x + i1, bad);
        rope_put(out + i0, quotient<POW2>((int64_t)cs.x * (int32_t)x0 - (int64_t)cs.y * (int32_t)x1, a.sf), bad);
        rope_put(out + i1, quotient<POW2>((int64_t)cs.y * (int32_t)x0 + (int64_t)cs.x * (int32_t)x1, a.sf), bad);
    }
    raise(a.flag, bad);
}

// The table of angles, a lane an entry: table[p][i] = the nearest integers to scale cos(p f_i), scale sin(p f_i), f_i = base^(-2 i / rot) slowed down by `factor` -- or, with
// `original` positions, a frequency that turns `high` times or more over them stays, one that turns `low` times or less is slowed down, those between in proportion.
// Correctly rounded operations in a fixed order (detmath.hpp): every device and host has the same table.
struct RopeTableArgs { double base, factor, original, low, high, scale; };
__global__ void __launch_bounds__(256) k_rope_table(int2* __restrict__ table, uint32_t rows, uint32_t pairs, const RopeTableArgs a) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (size_t)rows * pairs) return;
    const uint32_t p = (uint32_t)(id / pairs), i = (uint32_t)(id - (size_t)p * pairs);
    double f = zkd::exp_det(-((double)i / (double)pairs) * zkd::log_det(a.base));
    if (a.original > 0) {
        const double turns = a.original * f / 6.283185307179586476925;
        double keep = (turns - a.low) / (a.high - a.low);
        keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
        f = f * (keep + (1.0 - keep) / a.factor);
    } else f = f / a.factor;
    double s, c;
    zkd::sincos_det((double)p * f, &s, &c);
    table[id] = make_int2((int32_t)rint(c * a.scale), (int32_t)rint(s * a.scale));
}

// ---- field elements that stand for integers, rescaled twice, from [head][token][dim] to int32 [token][head][dim] ------------------------------------------------
__global__ void __launch_bounds__(256) k_i32_from_heads(int32_t* __restrict__ out, const Fr* __restrict__ in, uint32_t heads, uint32_t tokens, uint32_t dim, const Divisor first, const Divisor second,
                                                        uint32_t* __restrict__ flag) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (size_t)heads * tokens * dim) return;
    const size_t row = id / dim;
    const uint32_t j = (uint32_t)(id - row * dim);
    const uint32_t token = (uint32_t)(row / heads), head = (uint32_t)(row - (size_t)token * heads);
    int64_t v;
    uint32_t bad = 0;
    if (!fr_fits_i64(in[((size_t)head * tokens + token) * dim + j], v) || v > (1ll << 62) || v < -(1ll << 62)) { bad = ZK_VALUES_RANGE; v = 0; }
    v = first.shift >= 0 ? quotient<true>(v, first) : quotient<false>(v, first);
    v = second.shift >= 0 ? quotient<true>(v, second) : quotient<false>(v, second);
    out[id] = narrow(v, bad);
    raise(flag, bad);
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
    int pow2;                            // every divisor of the call is a power of two
    uint32_t* flag;
};
template <bool POW2> __device__ __forceinline__ uint32_t activation_at(int64_t g, const Epilogue& e, uint32_t& bad) {      // the place in the table, or the table's length
    const uint64_t at = (uint64_t)(quotient<POW2>(g, e.sf_gate) - e.low);
    bad |= at < e.len ? 0u : (uint32_t)ZK_VALUES_TABLE;
    return at < e.len ? (uint32_t)at : e.len;
}
template <bool POW2> __device__ __forceinline__ int32_t gated_value(int32_t act, int64_t u, const Epilogue& e, uint32_t& bad) {
    return narrow(quotient<POW2>((int64_t)act * narrow(quotient<POW2>(u, e.sf), bad), e.sf_hidden), bad);
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
    int64_t* parts;                      // a split contraction's sums, [part][weight][row][column]
    Epilogue e;
};
static constexpr uint32_t CHUNK = 256;
// sum_s a[s] 256^s: within -2^62 .. 2^62 - 1, or flagged and 0.  Six planes in all cannot leave that range: p digits hold 128 (256^p - 1) / 255 at most, and
// 43690 products of three by three digits, or of four by two, stay below 2^61.5.
template <int NS> __device__ __forceinline__ int64_t joined(const int32_t (&a)[NS], uint32_t& bad) {
    if constexpr (NS <= 5) {
        int64_t v = a[0];
#pragma unroll
        for (int s = 1; s < NS; ++s) v += (int64_t)a[s] << (8 * s);
        return v;
    } else {
        // |a[s]| < 2^31, so the two low terms are below 2^41 together, and the sum in units of 2^16, which the others' 2^56 leave room for, says whether it fits
        const int64_t lo = a[0] + (int64_t)a[1] * 256;
        int64_t hi = 0;
#pragma unroll
        for (int s = NS - 1; s >= 2; --s) hi = hi * 256 + a[s];
        const int64_t units = hi + (lo >> 16);
        const bool fits = (uint32_t)((int32_t)(units >> 32) + 0x4000) < 0x8000u;      // -2^46 .. 2^46 - 1
        bad |= fits ? 0u : (uint32_t)ZK_VALUES_RANGE;
        return fits ? (int64_t)((uint64_t)hi * 65536 + (uint64_t)lo) : 0;
    }
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
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0;
    if (row >= g.rows) return;
    const int32_t* p = g.x + row * g.ldx + k;
    if (g.x_aligned && k + 16 <= g.inner) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const v4i v = reinterpret_cast<const v4i*>(p)[w];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * w + e] = v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) if (k + e < g.inner) x[e] = p[e];
    }
}

// x's planes for the products of many rows.  A workgroup takes 32 rows and CHUNK columns, 32 columns of a wave's 64 at a time: a lane 16 values of a row, so that the
// wave writes 1 KB of every plane in one piece.  How many planes the stretch needs goes to a place of its own.  2048 x 4096: 14 us, 67 MB.
__global__ void __launch_bounds__(256) k_split_x(const ProductArgs g, int8_t* __restrict__ planes, uint32_t* __restrict__ need, v4i* __restrict__ zeros) {
    __shared__ uint32_t most[4];
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 64) zeros[threadIdx.x] = v4i{0, 0, 0, 0};
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.y * 32 + (lane >> 1), k0 = blockIdx.x * CHUNK + wave * 64 + 16 * (lane & 1u), Kp = g.w.Kp;
    uint32_t bad = 0, planes_needed = 1;
    int32_t x[2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i) row_piece(g, row, k0 + 32 * i, x[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (k0 + 32 * i >= Kp) break;          // Kp is a multiple of 128
        v4i d[4];
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) m = max(m, (uint32_t)(x[i][e] < 0 ? ~x[i][e] : x[i][e]));
        planes_needed = max(planes_needed, m <= 127u ? 1u : m <= 32639u ? 2u : m <= 8355711u ? 3u : 4u);      // p digits hold up to 127 (256^p - 1) / 255
        digit_planes(x[i], d, bad);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<v4i*>(planes + (size_t)j * g.rows_padded * Kp + plane_at(g.rows_padded, row, k0 + 32 * i)) = d[j];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) planes_needed = max(planes_needed, (uint32_t)__shfl_xor(planes_needed, off, 64));
    if (lane == 0) most[wave] = planes_needed;
    __syncthreads();
    if (threadIdx.x == 0) need[(size_t)blockIdx.y * g.chunks + blockIdx.x] = max(max(most[0], most[1]), max(most[2], most[3]));
    raise(g.e.flag, bad);
}

// What becomes of a tile's sums: outputs, by divisors that are powers of two or any, or parts of sums
enum class End { POW2, ANY, PARTS };
// Many rows.  A workgroup of four waves takes 64 MT rows by 64 NQ columns of weights -- with NQ = 2 64 of each where there are two: a wave's gate and up tiles lie in the same
// lanes, and what joins them needs no exchange -- and a wave 32 MT by 32 NQ, as 32 x 32 tiles of v_mfma_i32_32x32x32_i8.
// Steps of 32 contraction bytes go from memory to LDS without passing through registers, four buffers deep; a step's fragments are read while the step before
// is multiplied, since one wave a SIMD (256 accumulators with MT = 2) has nobody to cover for it.
// 2048 x 4096 x 4096, three planes by two: 156 us; both 4096 x 11008 weights at 2048 rows 860, 2.55 POP/s (the library's int8 product of 8192^3: 2.05).  The matrix units are
// busy 65 % of the cycles, at 1.75 to 1.85 GHz: the card's power holds the clock there (the same without the loads from memory, on what lies in LDS, 2.3 GHz and 570 us), and part of what
// saves stalls costs clock.  (The instructions alone, on random bytes, 129 us and 693 for these two, 3.2 POP/s.)  Steps of 64 bytes (61 us against 41 for 64 rows of 4096 x 11008 in tiles of 128 columns), eight buffers (47), the next tile's first steps ahead of a tile's outputs (936
// against 895 for the whole) and other orders of the products or tiles (within 1 %) gained nothing.
template <bool GATED, int PA, int PB, int MT, int NQ> struct Tile {
    static constexpr int NS = PA + PB - 1, TM = 64 * MT, TN = 64 * NQ, PIECES = PA * 2 * MT + PB * 2 * NQ, SHARE = (PIECES + 3) / 4, BYTES = (PA * TM + PB * TN) * 32;
    v16i acc[NS][MT][NQ];
    // steps first .. first + steps - 1 of the contraction, a multiple of four
    __device__ __forceinline__ void multiply(const ProductArgs& g, uint32_t m0, uint32_t n0, uint32_t first, uint32_t steps, int8_t* const (&buf)[4]) {
        const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), wm = wave >> 1, wn = wave & 1;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < NQ; ++q)
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
                const uint32_t cb = c - PA * 2 * MT, plane = cb / (2 * NQ), r = cb % (2 * NQ) * 32, row = n0 + (GATED ? r & 63u : r);
                const Planes& w = GATED && r < 64 ? g.gate : g.w;
                const bool has = (int)plane < w.n, inside = row < w.rows;
                src[i] = has ? w.p + (size_t)plane * w.rows * w.Kp + (size_t)(inside ? row : w.rows - 1) * 32 : g.zeros;
                at[i] = (has && inside ? min(lr, w.rows - 1 - row) : 0u) * 32 + lane_half;
                dst[i] = (PA * TM + plane * TN + r) * 32;
                step[i] = has ? (size_t)w.rows * 32 : 0;
            }
            src[i] += step[i] * first;
        }
        const uint32_t half = lane >> 5;
        const uint32_t rowA = wm * 32 * MT + (lane & 31), at_a = rowA * 32 + gemm_half(rowA, half) * 16;
        const uint32_t rowB = wn * (GATED ? 32 : 32 * NQ) + (lane & 31), next_b = GATED ? 64 : 32, at_b = (PA * TM + rowB) * 32 + gemm_half(rowB, half) * 16;      // 32 rows on: the same halves
        uint32_t fetched = 1;
        auto fetch = [&](int8_t* to) {                         // the next step; behind the last one that again, into buffers nobody reads any more
            const size_t on = (size_t)(int64_t)__builtin_amdgcn_readfirstlane(fetched < steps ? -1 : 0);
            ++fetched;
#pragma unroll
            for (int i = 0; i < SHARE; ++i) { load_to_lds(src[i] + at[i], to + dst[i]); src[i] += step[i] & on; }
        };
        struct Fragments { v4i a[PA][MT], b[PB][NQ]; };
        auto read = [&](const int8_t* from, Fragments& f) {
#pragma unroll
            for (int i = 0; i < PA; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m) f.a[i][m] = *reinterpret_cast<const v4i*>(from + at_a + (i * TM + 32 * m) * 32);
#pragma unroll
            for (int j = 0; j < PB; ++j)
#pragma unroll
                for (int q = 0; q < NQ; ++q) f.b[j][q] = *reinterpret_cast<const v4i*>(from + at_b + (j * TN + next_b * q) * 32);
        };
        auto products = [&](const Fragments& f) {
#pragma unroll
            for (int i = 0; i < PA; ++i)
#pragma unroll
                for (int j = 0; j < PB; ++j)
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int q = 0; q < NQ; ++q) acc[i + j][m][q] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[i][m], f.b[j][q], acc[i + j][m][q], 0, 0, 0);
        };
        // the fragments' reads and the next loads spread over the products
        auto spread = [&] {
            constexpr int READS = PA * MT + PB * NQ, PRODUCTS = PA * PB * MT * NQ;
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // an LDS read
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);      // a matrix instruction
            }
#pragma unroll
            for (int i = 0; i < SHARE; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);      // a load
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
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
        const std::integral_constant<int, 2> two;
        const std::integral_constant<int, 3> three;
        Fragments even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) fetch(buf[i]);
        arrived(three);
        read(buf[0], even);
        for (uint32_t t = 0; t < steps; t += 4) {
            arrived(two); fetch(buf[0]); read(buf[1], odd); products(even); spread();
            arrived(two); fetch(buf[1]); read(buf[2], even); products(odd); spread();
            arrived(two); fetch(buf[2]); read(buf[3], odd); products(even); spread();
            arrived(two); fetch(buf[3]); read(buf[0], even); products(odd); spread();
        }
        __builtin_amdgcn_s_waitcnt(7 << 4 | 15 << 8);          // vmcnt 0: no load into LDS outlives the workgroup or meets a next tile's
        __syncthreads();                                       // a next tile's loads find buffers that nobody reads any more
    }
    // The outputs, eight rows at a time: all their places in the table first, then the table's values, so that one wait covers them.  Stores go through a buffer
    // that ends with the last row, and a column beyond the last has no place in it.  (Such a column repeats the last and a row beyond the last is zeros: of the flags only the
    // table's needs to know.)
    template <End END> __device__ __forceinline__ void finish(const ProductArgs& g, uint32_t m0, uint32_t n0, uint32_t& bad) {
        constexpr bool POW2 = END == End::POW2;
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
        auto value = [&](int m, int q, int r) {
            int32_t a[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                a[s] = acc[s][m][q][r];
                asm("" : "+v"(a[s]));          // row by row: the compiler joins 16 rows at a time otherwise and spills
            }
            return joined<NS>(a, bad);
        };
        const uint32_t rows_here = m0 < g.rows ? min(g.rows - m0, (uint32_t)TM) : 0;
        if constexpr (END == End::PARTS) {
            const size_t weight = (size_t)g.rows * g.cols;
            int64_t* out = g.parts + (size_t)blockIdx.z * (GATED ? 2 : 1) * weight;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const uint32_t row = (wm * MT + m) * 32 + 4 * (lane >> 5) + 8 * (r >> 2) + (r & 3), col = n0 + (GATED ? wn * 32 : wn * 32 * NQ + q * 32) + (lane & 31);
                        const int64_t v = value(m, q, r);
                        if (row < rows_here && col < g.cols) out[(GATED ? q * weight : 0) + (size_t)(m0 + row) * g.cols + col] = v;
                    }
            return;
        }
        const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(g.e.out + (size_t)m0 * g.cols, 0, rows_here * g.cols * 4, 0x00027000);      // raw: plain bytes
        auto store = [&](uint32_t row, uint32_t col, int32_t y) { __builtin_amdgcn_raw_buffer_store_b32(y, out, n0 + col < g.cols ? (row * g.cols + n0 + col) * 4 : 0xFFFFFFFFu, 0, 0); };
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint32_t row0 = (wm * MT + m) * 32 + 4 * (lane >> 5);
            if constexpr (GATED) {
                const uint32_t col = wn * 32 + (lane & 31);
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += 8) {
                    uint32_t at[8];
                    int32_t act[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const uint32_t row = row0 + 8 * ((r0 + r) >> 2) + (r & 3);
                        uint32_t off = 0;
                        at[r] = activation_at<POW2>(value(m, 0, r0 + r), g.e, off);
                        bad |= row < rows_here ? off : 0u;
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) act[r] = g.e.table[min(at[r], g.e.len - 1)];
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        store(row0 + 8 * ((r0 + r) >> 2) + (r & 3), col, gated_value<POW2>(at[r] == g.e.len ? 0 : act[r], value(m, 1, r0 + r), g.e, bad));
                    __builtin_amdgcn_sched_barrier(0);         // the next rows' values would only crowd the registers
                }
            } else {
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        store(row0 + 8 * (r >> 2) + (r & 3), wn * 32 * NQ + q * 32 + (lane & 31), narrow(quotient<POW2>(value(m, q, r), g.e.sf), bad));
                        if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);      // the next rows' values would only crowd the registers
                    }
            }
        }
    }
};
template <bool GATED, int PB, int MT, int NQ, End END> __global__ void __launch_bounds__(256, MT == 2 || PB == 3 ? 1 : 2) k_product(const ProductArgs g) {
    constexpr int BYTES = Tile<GATED, 3, PB, MT, NQ>::BYTES > Tile<GATED, 4, PB, 1, NQ>::BYTES ? Tile<GATED, 3, PB, MT, NQ>::BYTES : Tile<GATED, 4, PB, 1, NQ>::BYTES;
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
    const uint32_t m0 = tm * 64 * MT, n0 = tn * (GATED ? 64 : 64 * NQ);
    uint32_t need = 0, bad = 0;
    for (uint32_t i = threadIdx.x & 63u; i < 2 * MT * g.chunks; i += 64) need = max(need, g.need[(size_t)(m0 / 32) * g.chunks + i]);
    const bool wide = __any(need > 3);
    const uint32_t fours = g.w.Kp / 128, first = END == End::PARTS ? fours * blockIdx.z / gridDim.z * 4 : 0, steps = END == End::PARTS ? fours * (blockIdx.z + 1) / gridDim.z * 4 - first : fours * 4;
    int8_t* const buf[4] = {s0, s1, s2, s3};
    if (!wide) {
        Tile<GATED, 3, PB, MT, NQ> t;
        t.multiply(g, m0, n0, first, steps, buf);
        t.template finish<END>(g, m0, n0, bad);
    } else {                                   // a value of more than three digits: all four planes, 64 rows at a time
        for (uint32_t m = m0; m < m0 + 64 * MT; m += 64) {
            Tile<GATED, 4, PB, 1, NQ> t;
            t.multiply(g, m, n0, first, steps, buf);
            t.template finish<END>(g, m, n0, bad);
        }
    }
    raise(g.e.flag, bad);
}

// The parts' sums added up, an output a lane: 64 rows of 4096 columns in four parts, 8 MB out of the caches, 4 us with its launch
template <bool GATED, bool POW2> __global__ void __launch_bounds__(256) k_product_join(const ProductArgs g, uint32_t parts) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, total = g.rows * g.cols;
    if (id >= total) return;
    constexpr int MATS = GATED ? 2 : 1;
    int64_t v[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) v[m] = 0;
    for (uint32_t p = 0; p < parts; ++p)
#pragma unroll
        for (int m = 0; m < MATS; ++m) v[m] += g.parts[((size_t)p * MATS + m) * total + id];
    uint32_t bad = 0;
    if constexpr (GATED) {
        const uint32_t at = activation_at<POW2>(v[0], g.e, bad);
        g.e.out[id] = gated_value<POW2>(at == g.e.len ? 0 : g.e.table[at], v[1], g.e, bad);
    } else g.e.out[id] = narrow(quotient<POW2>(v[0], g.e.sf), bad);
    raise(g.e.flag, bad);
}

// Few rows, or few tiles: the weights' way out of memory is what counts.  A workgroup takes 16 columns (of each weight) and 16 RT rows, its waves the units of 64 contraction
// bytes in turn, straight from memory into the fragments of v_mfma_i32_16x16x64_i8 -- a fragment of 16 columns is two pieces of 512 bytes in the planes' layout.
// SPLIT: x is split on the way, all four digits (one launch, and the matrix cores idle anyway); else its planes are read as the weights' are.  The waves'
// accumulators are added up in LDS, integers in any order.  One row of 11008 x 4096: 17.5 us, of both 4096 x 11008 weights 35, 5.15 TB/s of planes; 32 rows of
// 4096 x 11008 32 us, where x's planes, read anew by every strip, weigh as much as the weights.
template <bool GATED, int PB, int RT, int PA, bool SPLIT, int WAVES, int DEPTH> struct Strip {
    static constexpr int MATS = GATED ? 2 : 1, NS = PA + PB - 1, SUMS = NS * MATS * RT;
    static __device__ __forceinline__ void run(const ProductArgs& g, uint32_t strip, uint32_t row_block, int32_t (*sum)[256], uint32_t& bad) {
        const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = lane & 15u, q = lane >> 4;
        const uint32_t units = g.w.Kp / 64, col = min(strip * 16 + c, g.cols - 1), row0 = row_block * 16 * RT;
        for (uint32_t i = threadIdx.x; i < SUMS * 256; i += WAVES * 64) (&sum[0][0])[i] = 0;
        const int8_t* src[MATS][PB];
        const Planes* mats[2] = {GATED ? &g.gate : &g.w, &g.w};
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int j = 0; j < PB; ++j)
                src[m][j] = mats[m]->p + (size_t)(j < mats[m]->n ? j : 0) * mats[m]->rows * g.w.Kp + ((size_t)(q >> 1) * g.cols + col) * 32 + (q & 1u) * 16;
        const int8_t* px = g.px + ((size_t)(q >> 1) * g.rows_padded + row0 + c) * 32 + (q & 1u) * 16;
        const size_t w_step = (size_t)g.cols * 64, x_step = (size_t)g.rows_padded * 64, x_plane = (size_t)g.rows_padded * g.w.Kp;
        v4i acc[NS][MATS][RT];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[s][m][r] = v4i{0, 0, 0, 0};
        v4i w[DEPTH][MATS][PB], a[DEPTH][SPLIT ? 1 : RT][SPLIT ? 4 : PA];
        int32_t x[DEPTH][SPLIT ? RT : 1][16];
        auto load = [&](uint32_t u, int d) {
            u = min(u, units - 1);             // behind the last one that again: never multiplied
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int j = 0; j < PB; ++j) w[d][m][j] = *reinterpret_cast<const v4i*>(src[m][j] + u * w_step);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if constexpr (SPLIT) row_piece(g, row0 + r * 16 + c, u * 64 + q * 16, x[d][r]);
                else
#pragma unroll
                    for (int i = 0; i < PA; ++i) a[d][r][i] = *reinterpret_cast<const v4i*>(px + i * x_plane + u * x_step + r * 512);
            }
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
                        if constexpr (SPLIT) digit_planes(x[d][r], a[d][0], bad);
#pragma unroll
                        for (int i = 0; i < PA; ++i)
#pragma unroll
                            for (int j = 0; j < PB; ++j)
#pragma unroll
                                for (int m = 0; m < MATS; ++m)
                                    acc[i + j][m][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[d][SPLIT ? 0 : r][i], w[d][m][j], acc[i + j][m][r], 0, 0, 0);
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
        for (uint32_t i = threadIdx.x; i < RT * 256; i += WAVES * 64) {
            const uint32_t r = i >> 8, row = row0 + (i >> 4), out_col = strip * 16 + (i & 15u);
            if (row >= g.rows || out_col >= g.cols) continue;
            int64_t v[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                int32_t t[NS];
#pragma unroll
                for (int s = 0; s < NS; ++s) t[s] = sum[(s * MATS + m) * RT + r][i & 255u];
                v[m] = joined<NS>(t, bad);
            }
            auto value = [&](auto pow2) {
                constexpr bool POW2 = decltype(pow2)::value;
                if constexpr (GATED) {
                    const uint32_t at = activation_at<POW2>(v[0], g.e, bad);
                    return gated_value<POW2>(at == g.e.len ? 0 : g.e.table[at], v[1], g.e, bad);
                } else return narrow(quotient<POW2>(v[0], g.e.sf), bad);
            };
            g.e.out[(size_t)row * g.cols + out_col] = g.e.pow2 ? value(std::true_type()) : value(std::false_type());
        }
    }
};
template <bool GATED, int PB, int WAVES> __global__ void __launch_bounds__(64 * WAVES) k_product_row(const ProductArgs g) {
    using S = Strip<GATED, PB, 1, 4, true, WAVES, 4>;
    __shared__ int32_t sum[S::SUMS][256];
    uint32_t bad = 0;
    S::run(g, blockIdx.x, 0, sum, bad);
    raise(g.e.flag, bad);
}
template <bool GATED, int PB, int RT, int WAVES> __global__ void __launch_bounds__(64 * WAVES) k_product_strip(const ProductArgs g, uint32_t row_blocks) {
    constexpr int DEPTH = RT == 1 ? 4 : 2;
    using Three = Strip<GATED, PB, RT, 3, false, WAVES, DEPTH>;
    using Four = Strip<GATED, PB, RT, 4, false, WAVES, DEPTH>;
    __shared__ int32_t sum[Four::SUMS][256];
    // workgroups go to the eight dies in turn: a strip's row blocks follow each other on one die, whose L2 has its weights then
    const uint32_t slot = blockIdx.x >> 3, strip = slot / row_blocks * 8 + (blockIdx.x & 7u), row_block = slot % row_blocks;
    if (strip * 16 >= g.cols) return;
    uint32_t need = 0, bad = 0;
    for (uint32_t i = threadIdx.x & 63u; i < g.chunks; i += 64) need = max(need, g.need[(size_t)row_block * g.chunks + i]);
    if (!__any(need > 3)) Three::run(g, strip, row_block, sum, bad);
    else Four::run(g, strip, row_block, sum, bad);
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
    ZK_ARG(w->N <= MAX_INNER, std::string(name) + ": an inner dimension above 43690");
    ZK_ARG(w->planes != nullptr && w->pb >= 1 && w->pb <= 3, std::string(name) + ": the weight has elements beyond 8355711 (three digits of eight bits)");
    return 0;
}
static Planes planes_of(const MatmulRhs* w) { return Planes{(const int8_t*)w->planes, w->P, w->Kp, w->pb}; }

// Up to here a product is one launch that splits x itself: 16 rows of 4096 x 11008 40 us so and 28 with a launch of k_split_x before, 4 rows 24 and 28.
static constexpr uint32_t SPLIT_ROWS = 4;
static size_t padded_rows(uint32_t rows) { return ((size_t)rows + 127) / 128 * 128; }
// A long contraction with few tiles is split, so that every compute unit has a part of one: from 8192 on and for 33 rows and more, where neither strips nor tiles fill the card.
// 64 rows of 11008 x 4096 36 us (strips 48, whole tiles 81), 128 rows 52 (81), of both such weights 55 (75 in strips) and 77 (104); of 4096 x 4096 the second launch
// takes what the first gains (64 rows 19 either way, 128 rows 25 and 26; of two weights 34 and 28).  Two planes of weights: a part's sum stays in 64 bits then.
static constexpr size_t PARTS_BYTES = (size_t)16 << 20;
static bool may_split(uint32_t rows, uint32_t inner) { return rows > 32 && inner > 8064; }
static unsigned parts_of(const ProductArgs& g, size_t weights) {
    if (g.parts == nullptr) return 1;
    const size_t tiles = (size_t)cdiv(g.cols, 64) * cdiv(g.rows, 64), each = weights * g.rows * g.cols * sizeof(int64_t);
    return (unsigned)std::min<size_t>({256 / tiles, g.w.Kp / 512, PARTS_BYTES / each});
}
// Tiles of 128 rows where there is one for every compute unit (2048 x 4096 x 4096: 156 us, with 64 rows 165); a third plane of weights has no registers for that.
// Half as wide where every tile then finds a unit of its own (64 rows of 4096 x 11008, 86 tiles: 42 us and 36; 256 rows of 4096 x 4096, 128 tiles: 35 and 32; 384 rows, 192 tiles: 41 and 46).
template <bool GATED, int PB, bool POW2> static void launch_tiles(const ProductArgs& g, hipStream_t st) {
    constexpr End END = POW2 ? End::POW2 : End::ANY;
    const unsigned tn = cdiv(g.cols, GATED ? 64 : 128);
    if constexpr (PB == 2) if ((size_t)tn * cdiv(g.rows, 128) >= 256) {
        hipLaunchKernelGGL((k_product<GATED, PB, 2, 2, END>), dim3(tn, cdiv(g.rows, 128)), dim3(256), 0, st, g);
        return;
    }
    if constexpr (PB == 2) if (const unsigned parts = parts_of(g, GATED ? 2 : 1); parts > 1) {
        hipLaunchKernelGGL((k_product<GATED, PB, 1, GATED ? 2 : 1, End::PARTS>), dim3(cdiv(g.cols, 64), cdiv(g.rows, 64), parts), dim3(256), 0, st, g);
        hipLaunchKernelGGL((k_product_join<GATED, POW2>), dim3(cdiv((size_t)g.rows * g.cols, 256)), dim3(256), 0, st, g, parts);
        return;
    }
    if constexpr (!GATED) if ((size_t)tn * cdiv(g.rows, 64) <= 128) {
        hipLaunchKernelGGL((k_product<GATED, PB, 1, 1, END>), dim3(cdiv(g.cols, 64), cdiv(g.rows, 64)), dim3(256), 0, st, g);
        return;
    }
    hipLaunchKernelGGL((k_product<GATED, PB, 1, 2, END>), dim3(tn, cdiv(g.rows, 64)), dim3(256), 0, st, g);
}
// Strips of one row of tiles: with one for every compute unit at most, eight waves of a workgroup share its contraction; with more, four, and two workgroups of them lie on a
// unit, so that one's loads go on while the other adds up (one row of both 4096 x 11008 weights, 688 strips: 42 us with eight, 36 with four; of 11008 x 4096, 256
// strips: 17 and 20).
static constexpr unsigned STRIPS_EACH = 256;
template <bool GATED, int PB> static void launch_row(const ProductArgs& g, hipStream_t st) {
    const unsigned strips = cdiv(g.cols, 16);
    if (strips > STRIPS_EACH) hipLaunchKernelGGL((k_product_row<GATED, PB, 4>), dim3(strips), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_product_row<GATED, PB, 8>), dim3(strips), dim3(512), 0, st, g);
}
// Rows beyond SPLIT_ROWS.  Strips read every weight once for 16 or 32 rows, whatever their number; tiles make better use of what they read, but each takes a compute unit a
// sixth of a microsecond and more for 32 contraction bytes, however few there are, so the count of strips decides.  4096 x 4096, strips and tiles: 64 rows (512 strips) 19 us
// and 26, 96 rows (768) 24 and 26, 128 rows (1024) 28 and 26; 32 rows of 4096 x 11008 (688) 33 and 34, 64 rows (1376) 54 and 36.  Of both such weights, whose strips cost twice
// and whose tiles are no wider: 64 rows of 4096 x 4096 28 and 37, 96 rows 37 and 37, 32 rows of 4096 x 11008 57 and 51.
template <bool GATED, int PB> static void launch_product(const ProductArgs& g, hipStream_t st) {
    const unsigned row_blocks = cdiv(g.rows, 32), strips = (cdiv(g.cols, 16) + 7) / 8 * 8;
    if (g.rows <= 16) {
        if (strips > STRIPS_EACH) hipLaunchKernelGGL((k_product_strip<GATED, PB, 1, 4>), dim3(strips), dim3(256), 0, st, g, 1u);
        else hipLaunchKernelGGL((k_product_strip<GATED, PB, 1, 8>), dim3(strips), dim3(512), 0, st, g, 1u);
    } else if ((size_t)strips * row_blocks < (GATED ? 640u : 1024u) && !(PB == 2 && parts_of(g, GATED ? 2 : 1) > 1)) hipLaunchKernelGGL((k_product_strip<GATED, PB, 2, 8>), dim3(strips * row_blocks), dim3(512), 0, st, g, row_blocks);
    else if (g.e.pow2) launch_tiles<GATED, PB, true>(g, st);
    else launch_tiles<GATED, PB, false>(g, st);
}
template <bool GATED> static int product(const char* name, ProductArgs& g, void* flag_dev, void* workspace, size_t workspace_bytes, hipStream_t st) {
    ZK_ARG(g.x != nullptr && g.e.out != nullptr, std::string(name) + ": null tensor");
    ZK_ARG(g.x != g.e.out, std::string(name) + ": in place");
    ZK_ARG(g.ldx >= g.inner, std::string(name) + ": rows of x overlap (ldx below the inner dimension)");
    ZK_ARG(g.rows <= (1u << 18), std::string(name) + ": more than 262144 rows in one call");
    ZK_ARG(g.cols <= (1u << 22), std::string(name) + ": more than 4194304 columns");
    ZK_ARG(workspace == nullptr || workspace_bytes >= zk_i32_linear_workspace(g.rows, g.inner), std::string(name) + ": the workspace is smaller than zk_i32_linear_workspace says");
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    g.e.flag = flag.dev;
    g.x_aligned = (g.ldx & 3) == 0 && ((uintptr_t)g.x & 15) == 0;
    const int pb = std::max(g.w.n, GATED ? g.gate.n : 0);
    if (g.rows <= SPLIT_ROWS) {
        if (pb <= 2) launch_row<GATED, 2>(g, st);
        else launch_row<GATED, 3>(g, st);
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
    g.parts = may_split(g.rows, g.inner) ? (int64_t*)((char*)workspace + bytes - PARTS_BYTES) : nullptr;
    hipLaunchKernelGGL(k_split_x, dim3(g.chunks, g.rows_padded / 32), dim3(256), 0, st, g, (int8_t*)workspace, (uint32_t*)g.need, (v4i*)g.zeros);
    if (pb <= 2) launch_product<GATED, 2>(g, st);
    else launch_product<GATED, 3>(g, st);
    ZK_LAUNCH_CHECK();
    return flag.end(name);
}

template <int NV, int VEC, bool POW2, int THREADS> static void launch_norm_n(const NormArgs& a, uint32_t rows, hipStream_t st) {
    const unsigned threads = (unsigned)std::max<size_t>(64, ((size_t)cdiv(a.cols, NV * VEC) + 63) / 64 * 64);
    hipLaunchKernelGGL((k_residual_norm<NV, VEC, POW2, THREADS>), dim3(rows), dim3(threads), threads * VEC * sizeof(double), st, a);
}
// Four aligned columns a lane, once in its registers or, for many rows, twice, with half as many waves and streamed stores: 511 rows of 4096 10.3 us and 8.0, 1024 rows 16.9 and 12.9, 2048 rows 32.6 and
// 22.6; up to 256 rows both take no longer than the call, 8 us.  Rows of 1024 stay with the first (2048 of them 9.7 us and 8.0, 8192 28.4 and 21.5).  Four times up to 16384 columns: 1024 x 8192 35 us, where
// the kernel for rows of any length, which reads them again in every pass, takes 56 (2048 x 5120: 51 either way).  One column a lane where something is not aligned: 1024 x 4098 24 us.
template <bool POW2> static void launch_norm(const NormArgs& a, uint32_t rows, hipStream_t st) {
    auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    const bool vec = (a.cols & 3) == 0 && (a.ldx & 3) == 0 && (a.b == nullptr || (a.ldb & 3) == 0) && aligned(a.x) && aligned(a.b) && aligned(a.h) && aligned(a.n) && aligned(a.post) &&
                     aligned(a.gate) && aligned(a.w);
    if (vec && a.cols <= 4096 && (rows < 512 || a.cols <= 1024)) launch_norm_n<1, 4, POW2, 1024>(a, rows, st);
    else if (vec && a.cols <= 4096) launch_norm_n<2, 4, POW2, 512>(a, rows, st);
    else if (vec && a.cols <= 16384) launch_norm_n<4, 4, POW2, 1024>(a, rows, st);
    else if (!vec && a.cols <= 1024) launch_norm_n<1, 1, POW2, 1024>(a, rows, st);
    else if (!vec && a.cols <= 16384) launch_norm_n<16, 1, POW2, 1024>(a, rows, st);
    else hipLaunchKernelGGL(k_residual_norm_long<POW2>, dim3(rows), dim3(256), 0, st, a);
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
    ZK_ARG(cols <= (1u << 24), "zk_i32_residual_norm: rows of more than 2^24 columns");
    auto with_x = [&](const void* out) { return out == nullptr || rows == 1 || ((out != x || ldx == cols) && (out != b || ldb == cols)); };
    ZK_ARG(with_x(h) && with_x(n), "zk_i32_residual_norm: in place, rows must be cols apart");
    ZK_ARG(h == nullptr || h != n, "zk_i32_residual_norm: h and n are one tensor");
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, "zk_i32_residual_norm")) return rc;
    int e2 = 0;
    NormArgs a{(int32_t*)h, (int32_t*)n, (int32_t*)rms_inv, (const int32_t*)x, (const int32_t*)b, (const int32_t*)post, (const int32_t*)gate, (const int32_t*)w, ldx, ldb, 0, cols,
                     gate ? rows / gate_rows : 1, res, scale, eps, std::frexp(scale, &e2) == 0.5, divisor(sf), flag.dev};
    for (; a.row0 < rows; a.row0 += 1u << 20) {          // a launch has fewer than 2^32 lanes
        const uint32_t n_rows = std::min<uint32_t>(1u << 20, rows - (uint32_t)a.row0);
        if (a.sf.shift >= 0) launch_norm<true>(a, n_rows, st);
        else launch_norm<false>(a, n_rows, st);
    }
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
    ZK_ARG((uint64_t)heads * dim <= (1u << 30), std::string(name) + ": more than 2^30 elements a token");
    {
        const unsigned __int128 of_heads = (unsigned __int128)(heads - 1) * out_head + dim, of_tokens = (unsigned __int128)(tokens - 1) * out_token + dim;
        ZK_ARG(tokens == 1 || heads == 1 || out_token >= of_heads || out_head >= of_tokens, std::string(name) + ": the output's heads overlap (neither a token within the stride of heads nor a head within that of tokens)");
    }
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    // nothing rotated: no position is looked at, and every token's own number lies within 2^32 - 1
    const RopeArgs a{out, x, out_token, out_head, x_token, x_head, tokens, heads, dim, rot, neighbours, (const int2*)table, rot ? table_rows : 0xFFFFFFFFu, rot ? (const int32_t*)positions : nullptr,
                     rot ? first : 0, divisor(sf), flag.dev};
    const bool vec = !fr && rot % 8 == 0 && dim % 4 == 0 && ((out_token | out_head | x_token | x_head) & 3) == 0 && (((uintptr_t)out | (uintptr_t)x | (uintptr_t)table) & 15) == 0;
    const uint32_t units = heads * (vec ? rot / 8 + (dim - rot) / 4 : rot / 2 + (dim - rot));      // a token's
    const uint32_t step = std::max(1u, (1u << 30) / units);
    for (uint32_t t = 0; t < tokens; t += step) {
        const uint32_t total = std::min(step, tokens - t) * units;
        const dim3 grid(cdiv(total, 256)), block(256);
        if (fr) {
            if (a.sf.shift >= 0) hipLaunchKernelGGL((k_rope<Fr, 1, true>), grid, block, 0, st, a, t, total);
            else hipLaunchKernelGGL((k_rope<Fr, 1, false>), grid, block, 0, st, a, t, total);
        } else if (vec) {
            if (a.sf.shift >= 0) hipLaunchKernelGGL((k_rope<int32_t, 4, true>), grid, block, 0, st, a, t, total);
            else hipLaunchKernelGGL((k_rope<int32_t, 4, false>), grid, block, 0, st, a, t, total);
        } else {
            if (a.sf.shift >= 0) hipLaunchKernelGGL((k_rope<int32_t, 1, true>), grid, block, 0, st, a, t, total);
            else hipLaunchKernelGGL((k_rope<int32_t, 1, false>), grid, block, 0, st, a, t, total);
        }
        if (tokens - t <= step) break;
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

int zk_rope_table(void* table, uint32_t rows, uint32_t rot, double base, double factor, double original, double low, double high, double magnitude, uint32_t sf, void* stv) {
    if (rows == 0 || rot == 0) return 0;
    ZK_ARG(table != nullptr && rot % 2 == 0, "zk_rope_table: null table or an odd part of the head");
    ZK_ARG((size_t)rows * (rot / 2) <= 0x7FFFFFFFu, "zk_rope_table: more than 2^31 entries");
    ZK_ARG(base > 1 && base <= 1e15 && factor > 0 && factor >= 1e-6 && factor <= 1e6, "zk_rope_table: the base must lie above 1 (up to 1e15), the factor within 1e-6 .. 1e6");
    ZK_ARG((double)rows <= 2147483648.0 * std::min(factor, 1.0), "zk_rope_table: a last angle beyond 2^31");
    ZK_ARG(original == 0 || (original > 0 && original <= 1e15 && low >= 0 && high > low && high <= 1e15), "zk_rope_table: with original positions, 0 <= low < high");
    ZK_ARG(sf > 0 && magnitude > 0 && magnitude * (double)sf <= 1073741824.0, "zk_rope_table: scale times magnitude must lie within 2^30");
    hipLaunchKernelGGL(k_rope_table, dim3(cdiv((size_t)rows * (rot / 2), 256)), dim3(256), 0, (hipStream_t)stv, (int2*)table, rows, rot / 2,
                       RopeTableArgs{base, factor, original, low, high, magnitude * (double)sf});
    ZK_LAUNCH_CHECK();
    return 0;
}
int zk_i32_from_heads(void* out, const void* in, uint32_t heads, uint32_t tokens, uint32_t dim, uint32_t sf_first, uint32_t sf_second, void* flag_dev, void* stv) {
    if (heads == 0 || tokens == 0 || dim == 0) return 0;
    ZK_ARG(out != nullptr && in != nullptr && out != in, "zk_i32_from_heads: null tensor or in place");
    ZK_ARG(sf_first > 0 && sf_second > 0, "zk_i32_from_heads: a scaling factor of 0");
    ZK_ARG((unsigned __int128)heads * tokens * dim <= 0xFFFFFF00u, "zk_i32_from_heads: more elements than a tensor has");
    const size_t n = (size_t)heads * tokens * dim;
    hipStream_t st = (hipStream_t)stv;
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, "zk_i32_from_heads")) return rc;
    hipLaunchKernelGGL(k_i32_from_heads, dim3(cdiv(n, 256)), dim3(256), 0, st, (int32_t*)out, (const Fr*)in, heads, tokens, dim, divisor(sf_first), divisor(sf_second), flag.dev);
    ZK_LAUNCH_CHECK();
    return flag.end("zk_i32_from_heads");
}

int zk_i32_rhs_prepare(void** prepared, const void* B, uint32_t N, uint32_t P, void* stv) {
    hipStream_t st = (hipStream_t)stv;
    ZK_ARG(prepared != nullptr && B != nullptr && N > 0 && P > 0, "zk_i32_rhs_prepare: null argument or empty matrix");
    ZK_ARG(N <= MAX_INNER && P <= (1u << 22), "zk_i32_rhs_prepare: an inner dimension above 43690, or more than 4194304 columns");
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
    const hipError_t done = hipStreamSynchronize(st);         // B is the caller's again, and any stream may read the planes
    if (done != hipSuccess) { (void)pool_free(r->planes, st); return hip_fail(done, "hipStreamSynchronize", __FILE__, __LINE__); }
    *prepared = r.release();
    return 0;
}
size_t zk_i32_linear_workspace(uint32_t rows, uint32_t inner) {
    const size_t Kp = ((size_t)inner + GBK - 1) / GBK * GBK;
    if (rows <= SPLIT_ROWS) return 0;
    return padded_rows(rows) * Kp * 4 + 1024 + (padded_rows(rows) / 32 * ((Kp + CHUNK - 1) / CHUNK) * 4 + 15) / 16 * 16 + (may_split(rows, inner) ? PARTS_BYTES : 0);
}
int zk_i32_linear(void* out, const void* x, size_t ldx, const void* prepared, uint32_t rows, uint32_t sf, void* workspace, size_t workspace_bytes, void* flag_dev, void* stv) {
    const MatmulRhs* w = (const MatmulRhs*)prepared;
    if (const int rc = check_weight(w, "zk_i32_linear")) return rc;
    ZK_ARG(sf > 0, "zk_i32_linear: a scaling factor of 0");
    if (rows == 0) return 0;
    ProductArgs g{};
    g.x = (const int32_t*)x; g.ldx = ldx; g.rows = rows; g.inner = w->N; g.cols = w->P; g.w = planes_of(w);
    g.e.out = (int32_t*)out; g.e.sf = divisor(sf); g.e.pow2 = g.e.sf.shift >= 0;
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
    g.e.pow2 = g.e.sf.shift >= 0 && g.e.sf_gate.shift >= 0 && g.e.sf_hidden.shift >= 0;
    g.e.table = (const int32_t*)table; g.e.low = low; g.e.len = len;
    return product<true>("zk_i32_gated", g, flag_dev, workspace, workspace_bytes, (hipStream_t)stv);
}

}  // extern "C"
