// Digit planes: integer matrices as int8 matrices for the matrix cores.  Shared by the field products (matmul.hip) and the products of a
// layer's values (layer_kernels.hip).
#pragma once
#include <cstddef>
#include <cstdint>
#include <hip/hip_runtime.h>

namespace zk {

// Balanced base-256 digits of a small signed integer: x = sum_j d_j 256^j, d_j in [-128, 127].  Both operands are laid
// out as planes of rows along the contraction index, padded with zeros to a multiple of the GEMM's K tile Kp, A[b][m][k] in rows m of the
// planes b * pa + i and B[b][k][p], transposed on the way, in rows p of the planes b * pb + j.  A plane stands in blocks of 32 contraction
// bytes of all its rows (plane_at): every operand fragment of the matrix instruction is 16 consecutive bytes, and the 32 rows of a step
// that a wave brings to LDS at once are 1 KB in one piece.
__host__ __device__ __forceinline__ size_t plane_at(size_t rows, size_t row, uint32_t k) { return ((size_t)(k >> 5) * rows + row) * 32 + (k & 31u); }
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
static constexpr int GBK = 128;      // Kp is a multiple of this

// the balanced digits of a 32-bit integer, one a byte
__host__ __device__ __forceinline__ uint32_t digit_bytes(uint32_t x) { return (x + 0x80808080u) ^ 0x80808080u; }

static inline int digits_for(unsigned long long absmax) {      // planes needed for |x| <= absmax: p digits reach 127 (256^p - 1) / 255
    int p = 1;
    unsigned __int128 reach = 127;
    while (reach < absmax && p < 8) { reach = reach * 256 + 127; ++p; }
    return reach >= absmax ? p : 0;
}

// A right operand kept by the caller for many products (a layer's weight): its largest magnitude and, when it is a matrix of
// small integers, its digit planes in the GEMM's layout -- neither is computed again per product.  B: the field elements it was made from, null where it was made from int32.
struct MatmulRhs { const void* B = nullptr; uint32_t N = 0, P = 0, Kp = 0; unsigned long long mb = ~0ull; int pb = 0; void* planes = nullptr;
                   // a weight of 4 bits instead (zk_i32_rhs_prepare_q4): no planes, its codes, then the scales and zeros of `groups` groups of `group` rows
                   void* q4 = nullptr; uint32_t group = 0, groups = 0; };

// The two 16-byte halves of a row of 32 bytes change places every eight rows in LDS, so that the fragments' reads spread over all banks
__device__ __forceinline__ uint32_t gemm_half(uint32_t row, uint32_t h) { return h ^ ((row >> 3) & 1u); }
__device__ __forceinline__ void load_to_lds(const int8_t* src, int8_t* dst) {       // 16 bytes a lane, dst: the wave's first byte
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src, (__attribute__((address_space(3))) uint32_t*)dst, 16, 0, 0);
}

}  // namespace zk
