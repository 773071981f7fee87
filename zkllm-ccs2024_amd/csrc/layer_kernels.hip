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
#include "field.hpp"
#include "planes.hpp"
#include "rt.hpp"
#include "../../include/zkllm_hip.h"

using namespace zk;

// ---- quotients --------------------------------------------------------------------------------------------------------------------------
// shift >= 0: s is 2^shift, else any.  POW2 is a template argument where a kernel divides often: the general quotient is some 60 instructions.
struct Divisor { int64_t s, half; int shift; };
static Divisor divisor(uint32_t s) { return Divisor{(int64_t)s, (int64_t)(s >> 1), (s & (s - 1)) == 0 ? 31 - __builtin_clz(s) : -1}; }
__device__ __forceinline__ int64_t quotient_general(int64_t t, const Divisor& d) {      // |t| <= 2^62: the sum does not wrap
    const int64_t n = t + d.half, q = n / d.s;
    return q - (q * d.s > n ? 1 : 0);
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
// a weight's digit planes; a matrix of fewer planes than another reads zeros for the rest
struct Planes { const int8_t* p; uint32_t rows, Kp; int n; };
struct ProductArgs {
    const int32_t* x;
    size_t ldx;
    uint32_t rows, inner, cols;
    Planes w, gate;
    Epilogue e;
};
// 2^62 and beyond: flagged, so that what follows works on a sum that 64 bits hold
__device__ __forceinline__ int64_t checked_sum(__int128 v, uint32_t& bad) {
    if (v >= ((__int128)1 << 62) || v <= -((__int128)1 << 62)) { bad |= ZK_VALUES_RANGE; return 0; }
    return (int64_t)v;
}
// A lane an output, its weight's digits straight from the planes.
template <bool GATED> __global__ void __launch_bounds__(256) k_product_plain(const ProductArgs g) {
    const uint32_t col = blockIdx.x * 64 + (threadIdx.x & 63u), row = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (col >= g.cols || row >= g.rows) return;
    uint32_t bad = 0;
    const int32_t* x = g.x + row * g.ldx;
    auto dot = [&](const Planes& w) {
        int64_t acc[3] = {0, 0, 0};            // |x| < 2^31, a digit below 2^8, fewer than 2^17 of them
        for (int j = 0; j < 3; ++j) {
            if (j >= w.n) break;
            const int8_t* p = w.p + (size_t)j * w.rows * w.Kp;
            for (uint32_t k = 0; k < g.inner; ++k) acc[j] += (int64_t)x[k] * p[plane_at(w.rows, col, k)];
        }
        return checked_sum((__int128)acc[0] + ((__int128)acc[1] << 8) + ((__int128)acc[2] << 16), bad);
    };
    for (uint32_t k = 0; k < g.inner; ++k) if (x[k] > 0x7F7F7F7F) bad |= ZK_VALUES_RANGE;
    const int64_t v = dot(g.w);
    int32_t y;
    if constexpr (GATED) y = gated_value(dot(g.gate), v, g.e, bad);
    else y = narrow(quotient_any(v, g.e.sf), bad);
    g.e.out[(size_t)row * g.cols + col] = y;
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

template <bool GATED> static int product(const char* name, ProductArgs& g, void* flag_dev, void* workspace, size_t workspace_bytes, hipStream_t st) {
    ZK_ARG(g.x != nullptr && g.e.out != nullptr, std::string(name) + ": null tensor");
    ZK_ARG(g.ldx >= g.inner, std::string(name) + ": rows of x overlap (ldx below the inner dimension)");
    ZK_ARG(g.rows <= (1u << 18), std::string(name) + ": more than 262144 rows in one call");
    ZK_ARG(workspace == nullptr || workspace_bytes >= zk_i32_linear_workspace(g.rows, g.inner), std::string(name) + ": the workspace is smaller than zk_i32_linear_workspace says");
    CallFlag flag;
    if (const int rc = flag.begin(flag_dev, st, name)) return rc;
    g.e.flag = flag.dev;
    hipLaunchKernelGGL(k_product_plain<GATED>, dim3(cdiv(g.cols, 64), cdiv(g.rows, 4)), dim3(256), 0, st, g);
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
    return (size_t)rows * Kp * 4 + (((size_t)rows + 127) / 128 * 4 + 255) / 256 * 256;
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
