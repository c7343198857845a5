// 4-bit matrices with group scales: quantize, dequantize, and products with a few rows.
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
    const float want = zeros ? __fdiv_rn(__fsub_rn(hi, lo), 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f);
    const uint16_t bits = scale_bits(want, scale_f16);
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

// One warp an output channel of one row: lane l adds the bytes l, l + 32, ... of the row.
__global__ void __launch_bounds__(256) q4_matvec_simple_kernel(Q4Args a, int x_dtype) {
    const int lane = threadIdx.x & 31;
    const int64_t n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= a.N) return;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        int64_t e = 0;
        if (a.offsets) {
            if (r >= a.offsets[a.E]) return;
            int lo = 0, hi = a.E;  // offsets[lo] <= r < offsets[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (a.offsets[mid] <= r) lo = mid;
                else hi = mid;
            }
            e = lo;
        }
        const int64_t xr = a.row_map ? a.row_map[r] : r;
        float sum[2] = {0.f, 0.f};
        for (int p = 0; p < (a.up.data ? 2 : 1); ++p) {
            const Q4Mat &w = p ? a.up : a.w;
            for (int64_t b = lane; b < a.K / 2 && xr >= 0 && xr < a.x_rows; b += 32) {
                const int64_t sz = (e * (a.K / a.G) + 2 * b / a.G) * a.N + n;
                const int z = w.zeros ? w.zeros[sz] & 15 : 8;
                const int c = w.data[(e * a.N + n) * (a.K / 2) + b];
                const float t = (float)((c & 15) - z) * ld_act(a.x, xr * a.K + 2 * b, x_dtype) +
                                (float)((c >> 4) - z) * ld_act(a.x, xr * a.K + 2 * b + 1, x_dtype);
                sum[p] = fmaf(q4_scale(w.scales[sz], a.scale_f16), t, sum[p]);
            }
            sum[p] = warp_sum_f32(sum[p]);
        }
        if (lane == 0) {
            const float v = a.up.data ? swiglu_clamped(sum[0], sum[1], a.limit) : sum[0];
            st_act(a.y, r * a.N + n, v, a.y_dtype);
        }
    }
}

}  // namespace

int launch_q4_matvec(const Q4Args &a, int x_dtype, cudaStream_t st) {
    const int64_t rows = a.rows < 65535 ? a.rows : 65535;
    q4_matvec_simple_kernel<<<dim3((unsigned)cdiv(a.N, 8), (unsigned)rows), 256, 0, st>>>(a, x_dtype);
    VF_LAUNCH_CHECK("q4_matvec_simple_kernel");
    return VFMOE_OK;
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
