// 8-bit activation checkpoints: writing and reading them (format: mx8.h).
// A training step keeps every layer's output until its backward; at 440,000 x 300 that is 528 MB a layer in fp32 and 145 MB in this form.
// Both kernels are one pass over the data, bound by HBM: pack reads 4 (2) bytes a value and writes 1 + 1/32, unpack the reverse.  440,000 x 600 in
// fp32: 0.31 and 0.27 ms for 1.33 GB each, 4.3 and 4.8 TB/s (a large copy: 4.6).
#include "mx8.h"

#include <algorithm>

namespace geogcn {
namespace {

// A quad of columns per lane: 8 neighbouring lanes hold one block, whose maximum goes round them in three shuffles; a wave covers
// 8 blocks = 256 columns of a row and its stores (256 bytes of codes, 8 scale bytes) are contiguous.
template <typename T>
__global__ __launch_bounds__(256) void mx8_pack_kernel(int64_t n, int F, int qpr, const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ codes,
                                                       int64_t ldq, uint8_t* __restrict__ scale) {
    const int64_t total = n * qpr;                      // qpr: quads per row, a multiple of 8 (whole blocks)
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / qpr;
        const int c = (int)(q - r * qpr) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < F) {
            if constexpr (sizeof(T) == 4) x = *reinterpret_cast<const float4*>(X + r * ldx + c);
            else {
                const uint2 w = *reinterpret_cast<const uint2*>(X + r * ldx + c);
                x = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
            }
            x = mask4(x, c, F);
        }
        uint32_t m = max(max(mx8_abs_bits(x.x), mx8_abs_bits(x.y)), max(mx8_abs_bits(x.z), mx8_abs_bits(x.w)));
        m = max(m, (uint32_t)__shfl_xor((int)m, 1));
        m = max(m, (uint32_t)__shfl_xor((int)m, 2));
        m = max(m, (uint32_t)__shfl_xor((int)m, 4));
        const uint32_t b = mx8_scale_byte(m);
        *reinterpret_cast<uint32_t*>(codes + r * ldq + c) = mx8_encode4(x.x, x.y, x.z, x.w, mx8_inv_scale(b), b != 255u);
        if ((threadIdx.x & 7) == 0) scale[r * (ldq / kMxBlock) + c / kMxBlock] = (uint8_t)b;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void mx8_unpack_kernel(int64_t n, int F, int qpr, const uint8_t* __restrict__ codes, int64_t ldq,
                                                         const uint8_t* __restrict__ scale, T* __restrict__ Y, int64_t ldy) {
    const int64_t total = n * qpr;                      // qpr: quads per row of Y to write; the columns from F on are zero
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / qpr;
        const int c = (int)(q - r * qpr) * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < F) {
            y = mx8_decode4(*reinterpret_cast<const uint32_t*>(codes + r * ldq + c), mx8_scale(scale[r * (ldq / kMxBlock) + c / kMxBlock]));
            y = mask4(y, c, F);
        }
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(Y + r * ldy + c) = y;
        else *reinterpret_cast<uint2*>(Y + r * ldy + c) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
    }
}

int check_mx8(int64_t n, int32_t F, int32_t type, const void* X, int64_t ldx, const void* codes, int64_t ldq, const void* scale) {
    GEOGCN_REQUIRE(n >= 0 && F >= 0, GEOGCN_E_SIZE, "mx8: negative size");
    GEOGCN_REQUIRE(type == GEOGCN_T_F32 || type == GEOGCN_T_BF16, GEOGCN_E_ARG, "mx8: type %d is neither fp32 nor bf16", type);
    if (n == 0 || F == 0) return 0;
    GEOGCN_REQUIRE(X && codes && scale, GEOGCN_E_NULL, "mx8: null pointer");
    GEOGCN_REQUIRE(ldx >= (F + 3) / 4 * 4 && ldx % 4 == 0, GEOGCN_E_ALIGN, "mx8: pitch %lld of %d columns", (long long)ldx, F);
    GEOGCN_REQUIRE(ldq >= F && ldq % kMxBlock == 0, GEOGCN_E_ALIGN, "mx8: code pitch %lld of %d columns is not whole blocks", (long long)ldq, F);
    GEOGCN_REQUIRE(reinterpret_cast<uintptr_t>(X) % (type == GEOGCN_T_F32 ? 16 : 8) == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0,
                   GEOGCN_E_ALIGN, "mx8: base not aligned");
    return 0;
}

}  // namespace
}  // namespace geogcn

using namespace geogcn;

extern "C" int geogcn_mx8_pack(int64_t n, int32_t F, int32_t type, const void* X, int64_t ldx, uint8_t* codes, int64_t ldq, uint8_t* scale,
                               void* stream) {
    if (const int rc = check_mx8(n, F, type, X, ldx, codes, ldq, scale)) return rc;
    if (n == 0 || F == 0) return 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int qpr = (int)cdiv(F, kMxBlock) * (kMxBlock / 4);
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(n * qpr, 256), (int64_t)kNumCU * 32);
    if (type == GEOGCN_T_F32)
        hipLaunchKernelGGL(mx8_pack_kernel<float>, dim3(grid), dim3(256), 0, st, n, F, qpr, static_cast<const float*>(X), ldx, codes, ldq, scale);
    else
        hipLaunchKernelGGL(mx8_pack_kernel<uint16_t>, dim3(grid), dim3(256), 0, st, n, F, qpr, static_cast<const uint16_t*>(X), ldx, codes, ldq, scale);
    GEOGCN_LAUNCH_CHECK("mx8_pack_kernel");
    return 0;
}

extern "C" int geogcn_mx8_unpack(int64_t n, int32_t F, int32_t type, const uint8_t* codes, int64_t ldq, const uint8_t* scale, void* Y,
                                 int64_t ldy, void* stream) {
    if (const int rc = check_mx8(n, F, type, Y, ldy, codes, ldq, scale)) return rc;
    if (n == 0 || F == 0) return 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t pad = type == GEOGCN_T_F32 ? 4 : 64;             // pads kept zero: roundup4 (fp32), roundup64 (bf16), never past the pitch
    const int qpr = (int)(std::min<int64_t>(ldy, cdiv(F, pad) * pad) / 4);
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(n * qpr, 256), (int64_t)kNumCU * 32);
    if (type == GEOGCN_T_F32)
        hipLaunchKernelGGL(mx8_unpack_kernel<float>, dim3(grid), dim3(256), 0, st, n, F, qpr, codes, ldq, scale, static_cast<float*>(Y), ldy);
    else
        hipLaunchKernelGGL(mx8_unpack_kernel<uint16_t>, dim3(grid), dim3(256), 0, st, n, F, qpr, codes, ldq, scale, static_cast<uint16_t*>(Y), ldy);
    GEOGCN_LAUNCH_CHECK("mx8_unpack_kernel");
    return 0;
}
