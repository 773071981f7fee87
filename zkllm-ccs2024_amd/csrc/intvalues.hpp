// What the kernels over int32 tensors in fixed point share (layer_kernels.hip, decode_kernels.hip): quotients, flags, and digits of eight bits and their sums.
#pragma once
#include <cstring>
#include <memory>
#include <string>
#include "planes.hpp"
#include "rt.hpp"
#include "../../include/zkllm_hip.h"

namespace zk {

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

// ---- digits and sums of their products ----------------------------------------------------------------------------------------------
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
    int32_t most = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) most = max(most, x[e]);
    bad |= most > 0x7F7F7F7F ? (uint32_t)ZK_VALUES_RANGE : 0u;      // four digits reach no further
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = digit_bytes((uint32_t)x[4 * w + e]);
        const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), b = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
        const uint32_t c = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), e = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
        out[0][w] = (int)__builtin_amdgcn_perm(c, a, 0x05040100u);
        out[1][w] = (int)__builtin_amdgcn_perm(c, a, 0x07060302u);
        out[2][w] = (int)__builtin_amdgcn_perm(e, b, 0x05040100u);
        out[3][w] = (int)__builtin_amdgcn_perm(e, b, 0x07060302u);
    }
}

// ---- flags ---------------------------------------------------------------------------------------------------------------------------
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

}  // namespace zk
