// 4-bit matrices with group scales: quantize and dequantize (the products: q4_matvec.cuh).
#include "common.cuh"
#include "q4.h"

namespace vfmoe {

namespace {

__device__ __forceinline__ uint16_t scale_bits(float s, int f16) {
    return f16 ? __half_as_ushort(__float2half_rn(s)) : __bfloat16_as_ushort(__float2bfloat16_rn(s));
}

// One thread a group.  Without zero points s = max|w| / 7, q = round(w / s) + 8; with them s = (hi - lo) / 15 over
// the range extended to 0, z = round(-lo / s), q = round(w / s) + z.  The codes are made with the scale as it is
// stored (rounded to 16 bits), so that scale's rounding costs no more than the codes can follow.
__global__ void __launch_bounds__(128) q4_quantize_kernel(const void *__restrict__ src, int src_dtype, int64_t N,
                                                          int64_t K, int G, int64_t total, uint8_t *__restrict__ data,
                                                          uint16_t *__restrict__ scales, int scale_f16,
                                                          uint8_t *__restrict__ zeros) {
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int64_t groups = K / G;
    const int64_t g = i % groups, row = i / groups;       // row over all matrices
    const int64_t m = row / N, n = row % N;
    const int64_t at = row * K + g * G;
    float lo = 0.f, hi = 0.f;
    for (int j = 0; j < G; ++j) {
        const float v = ld_act(src, at + j, src_dtype);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    float want = __fdiv_rn(fmaxf(hi, -lo), 7.f);
    if (zeros) {
        const float range = __fsub_rn(hi, lo);  // of finite values, yet it may pass fp32
        want = isinf(range) ? __fsub_rn(__fdiv_rn(hi, 15.f), __fdiv_rn(lo, 15.f)) : __fdiv_rn(range, 15.f);
    }
    uint16_t bits = scale_bits(want, scale_f16);
    if (scale_f16 && bits == 0x7c00) bits = 0x7bff;  // past fp16: its largest value, an infinite scale would make zeros NaN
    const float s = q4_scale(bits, scale_f16);
    float z = 8.f;
    if (zeros) z = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 0.f;
    const int64_t sz = (m * groups + g) * N + n;
    scales[sz] = bits;
    if (zeros) zeros[sz] = (uint8_t)z;
    for (int j = 0; j < G; j += 2) {
        uint32_t b = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float v = ld_act(src, at + j + h, src_dtype);
            const float q = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(v, s)) + z, 0.f), 15.f) : z;
            b |= (uint32_t)q << (4 * h);
        }
        data[(at + j) / 2] = (uint8_t)b;
    }
}

// One thread a byte: its two values s * (q - z), one fp32 product each, rounded to the destination's type.
__global__ void __launch_bounds__(256) q4_dequant_kernel(Q4Mat w, int64_t N, int64_t K, int G, int64_t total,
                                                         int scale_f16, void *__restrict__ dst, int dst_dtype) {
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / (K / 2), k = 2 * (i % (K / 2));
    const int64_t sz = (row / N * (K / G) + k / G) * N + row % N;
    const float s = q4_scale(w.scales[sz], scale_f16);
    const int z = w.zeros ? w.zeros[sz] & 15 : 8;
    const int b = w.data[i];
    st_act(dst, 2 * i, s * (float)((b & 15) - z), dst_dtype);
    st_act(dst, 2 * i + 1, s * (float)((b >> 4) - z), dst_dtype);
}

}  // namespace

int launch_q4_matvec(const Q4Args &a, int x_dtype, cudaStream_t st) {
    return x_dtype == VFMOE_DT_BF16 ? launch_q4_bf16(a, st) : x_dtype == VFMOE_DT_F16 ? launch_q4_f16(a, st) : launch_q4_f32(a, st);
}

int launch_q4_quantize(const void *src, int src_dtype, int64_t N, int64_t K, int G, int64_t n_mats, uint8_t *data,
                       uint16_t *scales, int scale_f16, uint8_t *zeros, cudaStream_t st) {
    const int64_t total = n_mats * N * (K / G);
    q4_quantize_kernel<<<(unsigned)cdiv(total, 128), 128, 0, st>>>(src, src_dtype, N, K, G, total, data, scales,
                                                                   scale_f16, zeros);
    VF_LAUNCH_CHECK("q4_quantize_kernel");
    return VFMOE_OK;
}

int launch_q4_dequant(const Q4Mat &w, int64_t N, int64_t K, int G, int64_t n_mats, int scale_f16, void *dst,
                      int dst_dtype, cudaStream_t st) {
    const int64_t total = n_mats * N * (K / 2);
    q4_dequant_kernel<<<(unsigned)cdiv(total, 256), 256, 0, st>>>(w, N, K, G, total, scale_f16, dst, dst_dtype);
    VF_LAUNCH_CHECK("q4_dequant_kernel");
    return VFMOE_OK;
}

}  // namespace vfmoe
