// Products of 4-bit matrices with a few rows on the tensor cores (decode batches): y[r] = W x[r].
//
// W's codes are the m16n8k16 MMA's A operand, rows = output channels, and up to 8 NT rows of x its columns.  Per
// group of G elements the MMAs sum (q - z) x, both exact in the operand type (|q - z| <= 15; fp32 x goes as three bf16
// parts of 8 bits, each its own MMA), and the fp32 result is scaled once: y += s_g * part.
//
// What bounds it: W is read once, half a byte an element, so HBM; the second limit is the issue of the decode (11
// instructions for 8 codes of a 16-bit type), which is why a lane reads GB = G / 32 neighbouring words at a time, one set
// of scales serves GB steps, and MT tiles of 16 channels share the x fragments.
//
// A CTA owns 16 MT channels (16 with gate and up: one tile each) and one tile of rows.  Its 8 warps take K in chunks of
// 128 round robin, so each streams its own chunks of W, scales and x through its own shared-memory ring with cp.async,
// without a barrier among the warps; at the end the 8 partial sums are added in warp order (the result does not
// depend on the launch) and the epilogue rounds once.
//
// Any order of the elements within a step serves the product as long as both operands agree.  A word holds elements
// 8 w .. 8 w + 7; (word >> 4 i) & 0x000f000f is the pair (i, i + 4), so x's 8 elements are paired the same way.  Lane t of a
// quad takes the words t GB .. t GB + GB - 1 of a group, so all four lanes of an MMA lie in one group.
#pragma once

#include "common.cuh"
#include "q4.h"

namespace vfmoe {
namespace q4 {

constexpr int kWarps = 8;
constexpr int kChunk = 128;  // elements of K a warp takes at a time

__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The operand pairs (i, i + 4) of a word's codes less the zero point: base + q is exact with the code in the low bits
// of base (bf16 128, fp16 1024), and so is its difference from base + z (zc, both halves).
template <bool F16>
__device__ __forceinline__ void decode(uint32_t w, uint32_t zc, uint32_t (&a)[4]) {
    constexpr uint32_t base = F16 ? 0x64006400u : 0x43004300u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = ((w >> (4 * i)) & 0x000f000fu) | base;
        if constexpr (F16) {
            const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&t), *reinterpret_cast<const __half2 *>(&zc));
            a[i] = *reinterpret_cast<const uint32_t *>(&d);
        } else {
            const __nv_bfloat162 d =
                __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&t), *reinterpret_cast<const __nv_bfloat162 *>(&zc));
            a[i] = *reinterpret_cast<const uint32_t *>(&d);
        }
    }
}

// Places of 16-byte units in a warp's buffers, so that the fragment loads meet no bank twice.  W: 4 units a row of
// 64 bytes; a lane loads GB words, 8, 16 or 32 lanes at a time.  x (16-bit): 16 units a row; fp32: pairs of units
// (two lanes of a quarter warp share their banks).
template <int GB>
__device__ __forceinline__ int place_w(int row, int u) {
    return GB == 4 ? u : GB == 2 ? u ^ (((row >> 1) & 1) << 1) : u ^ ((row >> 1) & 3);
}
template <int GB>
__device__ __forceinline__ int place_x(int row, int u) {
    return GB == 4 ? u ^ ((u >> 3) & 1) ^ ((row & 1) << 1) : GB == 2 ? u ^ (row & 1) : u ^ ((row & 1) << 2);
}

// One lane's 8 elements of x as MMA B pairs: 16-bit types as they are, fp32 in three bf16 parts (truncated to 8 bits each:
// exact).  An infinity has no further parts, a NaN stays one.
template <int XD>
struct XFrag {
    static constexpr int kParts = XD == VFMOE_DT_F32 ? 3 : 1;
    uint32_t b[kParts][4];  // pairs (i, i + 4)
    // u: place of the unit (of the pair, fp32); zeros where the tile has no such row
    __device__ __forceinline__ void load(const uint8_t *row, int u, bool ok) {
        if constexpr (XD != VFMOE_DT_F32) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (ok) v = *reinterpret_cast<const uint4 *>(row + u * 16);
            b[0][0] = __byte_perm(v.x, v.z, 0x5410);
            b[0][1] = __byte_perm(v.x, v.z, 0x7632);
            b[0][2] = __byte_perm(v.y, v.w, 0x5410);
            b[0][3] = __byte_perm(v.y, v.w, 0x7632);
        } else {
            float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
            if (ok) {
                lo = *reinterpret_cast<const float4 *>(row + u * 32);
                hi = *reinterpret_cast<const float4 *>(row + u * 32 + 16);
            }
            const float e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            uint32_t part[3][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t h = __float_as_uint(e[i]);
                const bool finite = (h & 0x7f800000u) != 0x7f800000u;
                if (!finite && (h & 0x007fffffu)) h = 0x7fc00000u;
                const float m = finite ? e[i] - __uint_as_float(h & 0xffff0000u) : 0.f;
                part[0][i] = h;
                part[1][i] = __float_as_uint(m);
                part[2][i] = __float_as_uint(m - __uint_as_float(__float_as_uint(m) & 0xffff0000u));
            }
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) b[p][i] = __byte_perm(part[p][i], part[p][i + 4], 0x7632);
        }
    }
};

// Bytes of one warp's stage: W, scales, zero points, x rows.
template <int XD, int MT, int GB>
struct Stage {
    static constexpr int kGroups = 4 / GB;  // groups of a chunk
    static constexpr int kW = MT * 16 * 64;
    static constexpr int kS = kGroups * MT * 32;
    static constexpr int kZ = kGroups * MT * 16;
    static constexpr int kRow = XD == VFMOE_DT_F32 ? 512 : 256;
    __host__ __device__ static constexpr int bytes(int x_rows) { return kW + kS + kZ + x_rows * kRow; }
};

struct Tile {
    int64_t n0;            // first channel
    const uint8_t *w[2];   // rows n0 of the tile's matrices (gate and up, or W and its next 16 rows)
    const uint16_t *s[2];  // their scales and zero points: element g * N
    const uint8_t *z[2];
};

template <int XD, int NT, int MT, int GB, bool ACT, int S>
__global__ void __launch_bounds__(kWarps * 32) matvec_kernel(Q4Args a, int x_rows_max, int row_tiles) {
    using St = Stage<XD, MT, GB>;
    constexpr bool F16 = XD == VFMOE_DT_F16;
    constexpr int kParts = XFrag<XD>::kParts;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_row[8 * NT];  // rows of x of the tile, -1: none
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    // the matrix and its rows: blockIdx.y = a tile of rows (one matrix), or the y-th matrix that has rows
    int64_t e = 0, row0 = 0, row1 = a.rows;
    if (a.offsets) {
        int left = blockIdx.y;
        e = -1;
        for (int b = 0; b < a.E; b += 32) {
            const int i = b + lane;
            const int lo = i < a.E ? a.offsets[i] : 0, hi = i < a.E ? a.offsets[i + 1] : 0;
            unsigned m = __ballot_sync(0xffffffffu, hi > lo);
            if (left < __popc(m)) {
                for (; left > 0; --left) m &= m - 1;
                const int src = __ffs(m) - 1;
                e = b + src;
                row0 = __shfl_sync(0xffffffffu, lo, src);
                row1 = min((int64_t)__shfl_sync(0xffffffffu, hi, src), a.rows);
                break;
            }
            left -= __popc(m);
        }
        if (e < 0 || row0 < 0) return;
    } else {
        row0 = blockIdx.y * (int64_t)(8 * NT) * row_tiles;
        row1 = min(row0 + 8 * NT * row_tiles, a.rows);
    }

    const int64_t N = a.N, K = a.K, groups = K / a.G;
    Tile tl;
    tl.n0 = blockIdx.x * (int64_t)(ACT ? 16 : 16 * MT);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const Q4Mat &mat = ACT && m ? a.up : a.w;
        const int64_t n = min(tl.n0 + (ACT ? 0 : 16 * m), N - 16);  // a last tile past the end repeats its channels
        tl.w[m] = mat.data + (e * N + n) * (K / 2);
        tl.s[m] = mat.scales + e * groups * N + n;
        tl.z[m] = mat.zeros ? mat.zeros + e * groups * N + n : nullptr;
    }
    const bool has_z = a.w.zeros != nullptr;
    const int stage_bytes = St::bytes(x_rows_max);
    uint8_t *mine = smem + (int64_t)warp * S * stage_bytes;
    const int64_t chunks = (K + kChunk - 1) / kChunk;

    for (int64_t r0 = row0; r0 < row1; r0 += 8 * NT) {
        const int nr = (int)min((int64_t)(8 * NT), row1 - r0);
        if (tid < 8 * NT) {
            int64_t r = tid < nr ? (a.row_map ? a.row_map[r0 + tid] : r0 + tid) : -1;
            s_row[tid] = r >= 0 && r < a.x_rows ? (int)r : -1;
        }
        __syncthreads();

        auto fetch = [&](int64_t c, int stage) {
            uint8_t *buf = mine + stage * stage_bytes;
            const int64_t k0 = c * kChunk;
            const int kv = (int)min((int64_t)kChunk, K - k0);  // a multiple of 32
            // W: 16 MT rows of 4 units of 32 elements
            const int wr = lane >> 2, wu = lane & 3;
            if (wu * 32 < kv) {
#pragma unroll
                for (int i = 0; i < 2 * MT; ++i) {
                    const int row = wr + 8 * (i & 1);
                    cp16(buf + (i >> 1) * 1024 + row * 64 + place_w<GB>(row, wu) * 16,
                         tl.w[i >> 1] + row * (K / 2) + k0 / 2 + wu * 16);
                }
            }
            const int ng = kv / (GB * 32);
            const int64_t g0 = k0 / (GB * 32);
            {   // scales: two units a group and tile; zero points: one
                const int gi = lane / (2 * MT), m = lane / 2 % MT, h = lane & 1;
                if (gi < ng) cp16(buf + St::kW + gi * MT * 32 + m * 32 + h * 16, tl.s[m] + (g0 + gi) * N + h * 8);
            }
            if (has_z) {
                const int gi = lane / MT, m = lane % MT;
                if (gi < ng) cp16(buf + St::kW + St::kS + gi * MT * 16 + m * 16, tl.z[m] + (g0 + gi) * N);
            }
            // x: unit of 8 elements (two units of 16 bytes in fp32)
            constexpr int es = XD == VFMOE_DT_F32 ? 4 : 2;
            const int xu = lane & 15;
            if (xu * 8 < kv) {
                for (int row = lane >> 4; row < nr; row += 2) {
                    const int xr = s_row[row];
                    if (xr < 0) continue;
                    const uint8_t *src = reinterpret_cast<const uint8_t *>(a.x) + ((int64_t)xr * K + k0 + xu * 8) * es;
                    uint8_t *dst = buf + St::kW + St::kS + St::kZ + row * St::kRow + place_x<GB>(row, xu) * (8 * es);
                    cp16(dst, src);
                    if constexpr (XD == VFMOE_DT_F32) cp16(dst + 16, src + 16);
                }
            }
        };

        float acc[MT][NT][4] = {};
        bool ok[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) ok[j] = s_row[8 * j + g] >= 0;

#pragma unroll
        for (int s = 0; s < S - 1; ++s) {
            if (warp + s * (int64_t)kWarps < chunks) fetch(warp + s * (int64_t)kWarps, s);
            cp_commit();
        }
        int stage = 0;
        for (int64_t c = warp; c < chunks; c += kWarps) {
            cp_wait<S - 2>();
            __syncwarp();  // the stage is there for every lane, and every lane is done with the one before it
            {
                const int64_t next = c + (S - 1) * (int64_t)kWarps;
                const int into = stage == 0 ? S - 1 : stage - 1;
                if (next < chunks) fetch(next, into);
                cp_commit();
            }
            const uint8_t *buf = mine + stage * stage_bytes;
            const int ng = (int)min((int64_t)kChunk, K - c * kChunk) / (GB * 32);
            const uint8_t *xb = buf + St::kW + St::kS + St::kZ + g * St::kRow;
#pragma unroll
            for (int gi = 0; gi < St::kGroups; ++gi) {
                if (gi >= ng) break;
                uint32_t wd[MT][2][GB], zc[MT][2];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int row = g + 8 * h;
                        const uint8_t *src = buf + m * 1024 + row * 64;
                        if constexpr (GB == 4) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(src + t * 16);
                            wd[m][h][0] = v.x, wd[m][h][1] = v.y, wd[m][h][2] = v.z, wd[m][h][3] = v.w;
                        } else if constexpr (GB == 2) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(src + place_w<GB>(row, 2 * gi + (t >> 1)) * 16 +
                                                                            (t & 1) * 8);
                            wd[m][h][0] = v.x, wd[m][h][1] = v.y;
                        } else {
                            wd[m][h][0] = *reinterpret_cast<const uint32_t *>(src + place_w<GB>(row, gi) * 16 + t * 4);
                        }
                        const uint32_t z = has_z ? buf[St::kW + St::kS + gi * MT * 16 + m * 16 + row] & 15u : 8u;
                        zc[m][h] = (F16 ? 0x64006400u : 0x43004300u) + z * 0x00010001u;
                    }
                float part[MT][NT][4] = {};
#pragma unroll
                for (int j = 0; j < GB; ++j) {
                    uint32_t lo[MT][4], hi[MT][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        decode<F16>(wd[m][0][j], zc[m][0], lo[m]);
                        decode<F16>(wd[m][1][j], zc[m][1], hi[m]);
                    }
                    const int u = gi * 4 * GB + t * GB + j;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (NT > 1 && 8 * nt >= nr) break;
                        XFrag<XD> x;
                        x.load(xb + 8 * nt * St::kRow, place_x<GB>(g, u), ok[nt]);
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                mma<F16>(part[m][nt], lo[m][0], hi[m][0], lo[m][1], hi[m][1], x.b[p][0], x.b[p][1]);
                                mma<F16>(part[m][nt], lo[m][2], hi[m][2], lo[m][3], hi[m][3], x.b[p][2], x.b[p][3]);
                            }
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint16_t *sp = reinterpret_cast<const uint16_t *>(buf + St::kW + gi * MT * 32 + m * 32);
                    const float s0 = q4_scale(sp[g], a.scale_f16), s1 = q4_scale(sp[g + 8], a.scale_f16);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        acc[m][nt][0] = fmaf(s0, part[m][nt][0], acc[m][nt][0]);
                        acc[m][nt][1] = fmaf(s0, part[m][nt][1], acc[m][nt][1]);
                        acc[m][nt][2] = fmaf(s1, part[m][nt][2], acc[m][nt][2]);
                        acc[m][nt][3] = fmaf(s1, part[m][nt][3], acc[m][nt][3]);
                    }
                }
            }
            stage = stage == S - 1 ? 0 : stage + 1;
        }

        // the warps' sums, added in warp order: [warp][tile][lane][4]
        cp_wait<0>();
        __syncthreads();
        float4 *red = reinterpret_cast<float4 *>(smem);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                red[((warp * MT + m) * NT + nt) * 32 + lane] =
                    make_float4(acc[m][nt][0], acc[m][nt][1], acc[m][nt][2], acc[m][nt][3]);
        __syncthreads();
        constexpr int kOut = ACT ? 1 : MT;
        for (int i = tid; i < kOut * NT * 128; i += kWarps * 32) {
            const int ch = i & 15, tok = i / 16 % (8 * NT), m = i / (128 * NT);
            const int64_t n = tl.n0 + 16 * m + ch;
            if (tok >= nr || n >= N) continue;
            const int at = ((tok >> 3) * 32 + (ch & 7) * 4 + ((tok & 7) >> 1)) * 4 + (ch >> 3) * 2 + (tok & 1);
            const float *f = reinterpret_cast<const float *>(smem);
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                v[0] += f[(w * MT + m) * NT * 128 + at];
                if (ACT) v[1] += f[(w * MT + MT - 1) * NT * 128 + at];
            }
            st_act(a.y, (r0 + tok) * N + n, ACT ? swiglu_clamped(v[0], v[1], a.limit) : v[0], a.y_dtype);
        }
        __syncthreads();  // the buffers and s_row are used again
    }
}

// Launch with rows in tiles of 8 NT.
template <int XD, int NT, int MT, int GB, bool ACT, int S>
int launch_tile(const Q4Args &a, cudaStream_t st) {
    const int64_t most = a.rows < 8 * NT ? a.rows : 8 * NT;
    const int ring = kWarps * S * Stage<XD, MT, GB>::bytes((int)most);
    const int sums = kWarps * MT * NT * 128 * (int)sizeof(float);
    const int smem = ring > sums ? ring : sums;
    constexpr int kMost = kWarps * S * Stage<XD, MT, GB>::bytes(8 * NT);
    static_assert(kMost <= 227 * 1024 && kMost >= kWarps * MT * NT * 512, "shared memory");
    auto kernel = matvec_kernel<XD, NT, MT, GB, ACT, S>;
    const int rc = set_smem_attr_once(reinterpret_cast<const void *>(kernel), kMost);
    if (rc) return rc;
    const int64_t tiles = cdiv(a.rows, 8 * NT), per = cdiv(tiles, 65535);
    const dim3 grid((unsigned)cdiv(a.N, ACT ? 16 : 16 * MT),
                    (unsigned)(a.offsets ? (a.E < a.rows ? a.E : a.rows) : cdiv(tiles, per)));
    VF_CUDA(launch_pdl(kernel, grid, dim3(kWarps * 32), (size_t)smem, st, a, (int)most, (int)per));
    VF_LAUNCH_CHECK("q4 matvec_kernel");
    return VFMOE_OK;
}

template <int XD, int GB>
int launch_group(const Q4Args &a, cudaStream_t st) {
    // rows a tile: for sorted rows about twice the mean of the matrices that have some
    const int64_t mean = a.offsets ? cdiv(a.rows, a.E < a.rows ? a.E : a.rows) : a.rows;
    const int64_t want = a.offsets && a.rows > 8 ? 2 * mean : mean;
    constexpr bool F32 = XD == VFMOE_DT_F32;
    if (a.up.data) {
        if (want <= 8) return launch_tile<XD, 1, 2, GB, true, 3>(a, st);
        if (want <= 16 || F32) return launch_tile<XD, 2, 2, GB, true, F32 ? 2 : 3>(a, st);
        return launch_tile<XD, F32 ? 2 : 4, 2, GB, true, 2>(a, st);
    }
    if (want <= 8) {
        if (a.N <= 32 * 148) return launch_tile<XD, 1, 1, GB, false, 3>(a, st);
        return launch_tile<XD, 1, 2, GB, false, 3>(a, st);
    }
    if (want <= 16 || F32) return launch_tile<XD, 2, 2, GB, false, F32 ? 2 : 3>(a, st);
    return launch_tile<XD, F32 ? 2 : 4, 2, GB, false, 2>(a, st);
}

template <int XD>
int launch_type(const Q4Args &a, cudaStream_t st) {
    return a.G == 32 ? launch_group<XD, 1>(a, st) : a.G == 64 ? launch_group<XD, 2>(a, st) : launch_group<XD, 4>(a, st);
}

}  // namespace q4
}  // namespace vfmoe
