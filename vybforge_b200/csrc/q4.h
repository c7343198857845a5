// 4-bit matrices with group scales: launch interface between api.cu and q4.cu / q4_matvec.cuh.
#pragma once

#include "common.cuh"

namespace vfmoe {

// n_mats matrices [N][K] (rows = output channels), w = s * (q - z):
//   data    codes, two a byte, element 2j of a row in the low nibble of byte j: [n_mats][N][K/2]
//   scales  [n_mats][K/G][N], fp16 or bf16
//   zeros   [n_mats][K/G][N], one byte each (low four bits count); 0: every zero point is 8
struct Q4Mat {
    const uint8_t *data;
    const uint16_t *scales;
    const uint8_t *zeros;
};

struct Q4Args {
    int64_t N, K;
    int G, E;
    int scale_f16;         // scales are fp16 (else bf16)
    Q4Mat w, up;           // up.data != 0: y = silu(min(w x, limit)) * clip(up x, -limit, limit)
    float limit;
    const void *x;         // [x_rows][K]
    int64_t x_rows;
    const int32_t *row_map;  // row of x of each output row, or 0
    const int32_t *offsets;  // [E + 1]: matrix e's rows are [offsets[e], offsets[e+1]), or 0 (one matrix)
    int64_t rows;          // output rows (a bound where offsets are given)
    void *y;               // [rows][N]
    int y_dtype;
};

int launch_q4_matvec(const Q4Args &a, int x_dtype, cudaStream_t st);
// one translation unit a type of x (q4_bf16.cu, q4_f16.cu, q4_f32.cu)
int launch_q4_bf16(const Q4Args &a, cudaStream_t st);
int launch_q4_f16(const Q4Args &a, cudaStream_t st);
int launch_q4_f32(const Q4Args &a, cudaStream_t st);
int launch_q4_quantize(const void *src, int src_dtype, int64_t N, int64_t K, int G, int64_t n_mats, uint8_t *data,
                       uint16_t *scales, int scale_f16, uint8_t *zeros, cudaStream_t st);
int launch_q4_dequant(const Q4Mat &w, int64_t N, int64_t K, int G, int64_t n_mats, int scale_f16, void *dst,
                      int dst_dtype, cudaStream_t st);

__device__ __forceinline__ float q4_scale(uint16_t s, int f16) {
    return f16 ? __half2float(__ushort_as_half(s)) : __uint_as_float((uint32_t)s << 16);
}

}  // namespace vfmoe
