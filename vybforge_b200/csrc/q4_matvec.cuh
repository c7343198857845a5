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
// A CTA owns 16 MT channels (16 with gate and up: one tile each) and one tile of rows.  Its warps take K in chunks of
// 128 round robin, so each streams its own chunks of W, scales and x through its own shared-memory ring with cp.async,
// without a barrier among the warps; at the end the partial sums are added in warp order (the result does not
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

#ifndef Q4W
#define Q4W 4
#define Q4C 4
#define Q4B 1000
#define Q4S 2
#endif
constexpr int kWarps = Q4W;
constexpr int kCtas = Q4C;
constexpr int kChunk = 128;  // elements of K a warp takes at a time

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Zero points as decode() takes them: base + z, and for fp16 also -(64 + z), in both halves.
template <bool F16>
struct Zero {
    uint32_t c, d;
    __device__ __forceinline__ explicit Zero(uint32_t z)
        : c((F16 ? 0x64006400u : 0x43004300u) + z * 0x00010001u), d(0xd400d400u + z * 0x00100010u) {}
};

// The operand pairs (i, i + 4) of a word's codes less the zero point: base + q is exact with the code in the low bits of
// base (bf16 128, fp16 1024), and so is its difference from base + z.  fp16 has room for the code four bits up: 1024 + 16 q,
// and (1024 + 16 q) / 16 - (64 + z) is one exact fma, which saves two of the three shifts.  Shifts and masks run on the
// ALU pipe at half the rate of the others, so they, not the subtractions, are what this kernel counts.
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(v), "r"(mask), "r"(base));
    return d;
}

template <bool F16>
__device__ __forceinline__ void decode(uint32_t w, const Zero<F16> &z, uint32_t (&a)[4]) {
    if constexpr (F16) {
        const __half2 c = *reinterpret_cast<const __half2 *>(&z.c), d = *reinterpret_cast<const __half2 *>(&z.d);
        const __half2 r = __float2half2_rn(0.0625f);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t v = i ? w >> 8 : w;
            const uint32_t t0 = and_or(v, 0x000f000fu, 0x64006400u), t1 = and_or(v, 0x00f000f0u, 0x64006400u);
            const __half2 q0 = __hsub2(*reinterpret_cast<const __half2 *>(&t0), c);
            const __half2 q1 = __hfma2(*reinterpret_cast<const __half2 *>(&t1), r, d);
            a[i] = *reinterpret_cast<const uint32_t *>(&q0);
            a[i + 1] = *reinterpret_cast<const uint32_t *>(&q1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
            const __nv_bfloat162 q =
                __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&t), *reinterpret_cast<const __nv_bfloat162 *>(&z.c));
            a[i] = *reinterpret_cast<const uint32_t *>(&q);
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

// 8 elements of x as MMA B pairs (i, i + 4): a 16-bit type as it is, fp32 in three bf16 parts (cut to 8 bits each: exact).
// An infinity has no further parts, a NaN stays one.
__device__ __forceinline__ uint4 pairs16(uint4 v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}
__device__ __forceinline__ void pairs32(uint4 lo, uint4 hi, uint4 (&out)[3]) {
    const uint32_t e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t part[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t h = e[i];
        const bool finite = (h & 0x7f800000u) != 0x7f800000u;
        if (!finite && (h & 0x007fffffu)) h = 0x7fc00000u;
        const float m = finite ? __uint_as_float(h) - __uint_as_float(h & 0xffff0000u) : 0.f;
        part[0][i] = h;
        part[1][i] = __float_as_uint(m);
        part[2][i] = __float_as_uint(m - __uint_as_float(__float_as_uint(m) & 0xffff0000u));
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
        out[p] = make_uint4(__byte_perm(part[p][0], part[p][4], 0x7632), __byte_perm(part[p][1], part[p][5], 0x7632),
                            __byte_perm(part[p][2], part[p][6], 0x7632), __byte_perm(part[p][3], part[p][7], 0x7632));
}

// Bytes of one warp's stage: W, scales, zero points, x rows.  HELD (one or two rows): x goes through a lane's
// registers and is kept as MMA pairs; else it is copied as it lies in memory, and every use pairs it.
template <int XD, int NT, int MT, int GB, bool HELD>
struct Stage {
    static constexpr int kGroups = 4 / GB;  // groups of a chunk
    static constexpr int kW = MT * 16 * 64;
    static constexpr int kS = kGroups * MT * 32;
    static constexpr int kZ = kGroups * MT * 16;
    static constexpr int kRow = XD != VFMOE_DT_F32 ? 256 : HELD ? 768 : 512;
    __host__ __device__ static constexpr int bytes(int x_rows) { return kW + kS + kZ + x_rows * kRow; }
};

template <int XD, int NT, int MT, int GB, bool ACT, bool SF16, bool HELD, int S>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? kCtas : 3) matvec_kernel(Q4Args a, int x_rows_max, int row_tiles) {
    using St = Stage<XD, NT, MT, GB, HELD>;
    constexpr int kTile = HELD ? 2 : 8 * NT;  // rows of x at a time
    constexpr bool F16 = XD == VFMOE_DT_F16, F32 = XD == VFMOE_DT_F32;
    constexpr int kParts = F32 ? 3 : 1;
    constexpr int es = F32 ? 4 : 2;
    constexpr int kTiles = ACT ? MT / 2 : MT;  // tiles of 16 channels of y
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_x[8 * NT];                // byte offset of the tile's rows in x, -1: none
    __shared__ __align__(128) uint8_t s_zero[St::kRow];  // what lanes without a row read
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    for (int i = tid * 4; i < St::kRow; i += kWarps * 128) *reinterpret_cast<uint32_t *>(s_zero + i) = 0u;

    // the matrix and its rows: blockIdx.y = a run of row tiles (one matrix), or the y-th matrix that has rows
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
        row0 = blockIdx.y * (int64_t)kTile * row_tiles;
        row1 = min(row0 + (int64_t)kTile * row_tiles, a.rows);
    }

    const int64_t N = a.N, n0 = blockIdx.x * (int64_t)(16 * kTiles);
    const int K = (int)a.K, groups = K / (32 * GB), chunks = (K + kChunk - 1) / kChunk;
    const bool has_z = a.w.zeros != nullptr;
    // MMA tile m: gate and up alternate; a last tile past the end repeats the last 16 channels
    auto channel = [&](int m) { return min(n0 + 16 * (ACT ? m >> 1 : m), N - 16); };
    auto matrix = [&](int m) -> const Q4Mat & { return ACT && (m & 1) ? a.up : a.w; };
    // what this lane copies of the warp's first chunk: 16 bytes of rows wr and wr + 8 of each tile, of the scales of
    // one tile and group, of the zero points of one, and of each second row of x
    const int wr = lane >> 2, wu = lane & 3;
    const uint8_t *w_src[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
        w_src[m] = matrix(m).data + (e * N + channel(m) + wr) * (K / 2) + warp * (kChunk / 2) + wu * 16;
    const int64_t w_next = 4 * (int64_t)K;  // 8 rows down
    const int sg = lane / (2 * MT), sm = lane / 2 % MT, zg = lane / MT, zm = lane % MT;
    const int g0 = warp * St::kGroups;
    const uint16_t *s_src = matrix(sm).scales + (e * groups + g0 + sg) * N + channel(sm) + (lane & 1) * 8;
    const uint8_t *z_src = has_z ? matrix(zm).zeros + (e * groups + g0 + zg) * N + channel(zm) : nullptr;
    const int64_t sz_step = (int64_t)kWarps * St::kGroups * N;
    const int xu = lane & 15;
    const uint8_t *x_src = reinterpret_cast<const uint8_t *>(a.x) + (warp * kChunk + xu * 8) * es;

    const int stage_bytes = St::bytes(x_rows_max);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S * stage_bytes;
    uint8_t *const mine = smem + warp * S * stage_bytes;
    constexpr int kX = St::kW + St::kS + St::kZ;  // x within a stage
    const uint32_t w_dst = ring + wr * 64 + place_w<GB>(wr, wu) * 16;
    const uint32_t s_dst = ring + St::kW + sg * MT * 32 + sm * 32 + (lane & 1) * 16;
    const uint32_t z_dst = ring + St::kW + St::kS + zg * MT * 16 + zm * 16;
    static_assert(St::kGroups * MT * 2 <= 32, "one copy of scales a lane");

    for (int64_t r0 = row0; r0 < row1; r0 += kTile) {
        const int nr = (int)min((int64_t)kTile, row1 - r0);
        if (tid < 8 * NT) {
            const int64_t r = tid < nr ? (a.row_map ? a.row_map[r0 + tid] : r0 + tid) : -1;
            s_x[tid] = r >= 0 && r < a.x_rows ? r * K * es : -1;
        }
        __syncthreads();

        // W, scales and zero points of the warp's i-th chunk (chunk warp + i * kWarps of the row) into a stage
        auto fetch_w = [&](int i, uint32_t at, int kv) {  // kv: elements left, a multiple of 32
            if (wu * 32 < kv) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint8_t *src = w_src[m] + (int64_t)i * (kWarps * kChunk / 2);
                    cp16(w_dst + at + m * 1024, src);
                    cp16(w_dst + at + m * 1024 + 512, src + w_next);
                }
            }
            if (sg < St::kGroups && sg * GB * 32 < kv) cp16(s_dst + at, s_src + i * sz_step);
            if (has_z && zg < St::kGroups && zg * GB * 32 < kv) cp16(z_dst + at, z_src + i * sz_step);
        };
        // x, at most two rows: lane l holds unit l % 16 of row l / 16
        uint4 held[F32 ? 2 : 1];
        const int64_t x_off = HELD && (lane >> 4) < nr ? s_x[lane >> 4] : -1;
        auto load_x = [&](int i, int kv) {
            if (x_off >= 0 && xu * 8 < kv) {
                const uint4 *src = reinterpret_cast<const uint4 *>(x_src + x_off + (int64_t)i * (kWarps * kChunk * es));
                held[0] = __ldg(src);
                if constexpr (F32) held[1] = __ldg(src + 1);
            }
        };
        auto store_x = [&](uint8_t *buf, int kv) {
            if (x_off >= 0 && xu * 8 < kv) {
                const int row = lane >> 4;
                uint8_t *dst = buf + kX + row * St::kRow + place_x<GB>(row, xu) * 16;
                if constexpr (F32) {
                    uint4 p[3];
                    pairs32(held[0], held[1], p);
#pragma unroll
                    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4 *>(dst + 256 * q) = p[q];
                } else {
                    *reinterpret_cast<uint4 *>(dst) = pairs16(held[0]);
                }
            }
        };
        // x, more rows
        auto fetch_x = [&](int i, uint32_t at, int kv) {
            if (xu * 8 < kv) {
#pragma unroll
                for (int j = 0; j < 4 * NT; ++j) {
                    if (2 * j >= nr) break;
                    const int row = 2 * j + (lane >> 4);
                    const int64_t off = s_x[row];
                    if (off < 0) continue;
                    const uint8_t *src = x_src + off + (int64_t)i * (kWarps * kChunk * es);
                    const uint32_t dst = ring + at + kX + row * St::kRow + place_x<GB>(row, xu) * (8 * es);
                    cp16(dst, src);
                    if constexpr (F32) cp16(dst + 16, src + 16);
                }
            }
        };

        float acc[MT][NT][4] = {};
        bool ok[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) ok[j] = 8 * j + g < kTile && s_x[8 * j + g] >= 0;

        const int runs = (chunks - warp + kWarps - 1) / kWarps;  // chunks of this warp
        const int left0 = K - warp * kChunk;                     // elements from its first chunk on
        constexpr int kStep = kWarps * kChunk;
#pragma unroll
        for (int i = 0; i < S - 1; ++i) {
            if (i < runs) {
                fetch_w(i, i * stage_bytes, left0 - i * kStep);
                if constexpr (!HELD) fetch_x(i, i * stage_bytes, left0 - i * kStep);
            }
            cp_commit();
        }
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (i < runs) {
                    load_x(i, left0 - i * kStep);
                    store_x(mine + i * stage_bytes, left0 - i * kStep);
                }
            if (S - 1 < runs) load_x(S - 1, left0 - (S - 1) * kStep);
        }
        int stage = 0;
        for (int i = 0; i < runs; ++i) {
            cp_wait<S - 2>();
            __syncwarp();  // the stage is there for every lane, and every lane is done with the one before it
            const int kv = left0 - i * kStep;
            if (i + S - 1 < runs) {
                const int into = (stage == 0 ? S - 1 : stage - 1) * stage_bytes;
                const int kn = kv - (S - 1) * kStep;
                fetch_w(i + S - 1, into, kn);
                if constexpr (HELD) {
                    store_x(mine + into, kn);
                    if (i + S < runs) load_x(i + S, kn - kStep);
                } else {
                    fetch_x(i + S - 1, into, kn);
                }
            }
            cp_commit();
            const uint8_t *buf = mine + stage * stage_bytes;
            stage = stage == S - 1 ? 0 : stage + 1;
            const uint8_t *xb[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) xb[nt] = ok[nt] ? buf + kX + (8 * nt + g) * St::kRow : s_zero;
#pragma unroll
            for (int gi = 0; gi < St::kGroups; ++gi) {
                if (gi * GB * 32 >= kv) break;
                // the words of channel row g + 8 h of tile m
                auto words = [&](int m, int h, uint32_t (&wd)[GB]) {
                    const uint8_t *src = buf + m * 1024 + h * 512 + g * 64;
                    if constexpr (GB == 4) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(src + t * 16);
                        wd[0] = v.x, wd[1] = v.y, wd[2] = v.z, wd[3] = v.w;
                    } else if constexpr (GB == 2) {
                        const uint2 v =
                            *reinterpret_cast<const uint2 *>(src + place_w<GB>(g, 2 * gi + (t >> 1)) * 16 + (t & 1) * 8);
                        wd[0] = v.x, wd[1] = v.y;
                    } else {
                        wd[0] = *reinterpret_cast<const uint32_t *>(src + place_w<GB>(g, gi) * 16 + t * 4);
                    }
                };
                auto x_pairs = [&](int nt, int j, uint4 (&xp)[kParts]) {
                    const int u = place_x<GB>(g, gi * 4 * GB + t * GB + j);
                    if constexpr (HELD) {
#pragma unroll
                        for (int p = 0; p < kParts; ++p) xp[p] = *reinterpret_cast<const uint4 *>(xb[nt] + 256 * p + u * 16);
                    } else if constexpr (F32) {
                        const uint4 *src = reinterpret_cast<const uint4 *>(xb[nt] + u * 32);
                        pairs32(src[0], src[1], xp);
                    } else {
                        xp[0] = pairs16(*reinterpret_cast<const uint4 *>(xb[nt] + u * 16));
                    }
                };
                const uint8_t *zp = buf + St::kW + St::kS + gi * MT * 16 + g;
                auto step = [&](const uint32_t (&lo)[4], const uint32_t (&hi)[4], const uint4 (&xp)[kParts], float (&part)[4]) {
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        mma<F16>(part, lo[0], hi[0], lo[1], hi[1], xp[p].x, xp[p].y);
                        mma<F16>(part, lo[2], hi[2], lo[3], hi[3], xp[p].z, xp[p].w);
                    }
                };
                auto scale = [&](int m, const float (&part)[4], float (&sum)[4]) {
                    const uint16_t *sp = reinterpret_cast<const uint16_t *>(buf + St::kW + gi * MT * 32 + m * 32);
                    const float s0 = q4_scale(sp[g], SF16), s1 = q4_scale(sp[g + 8], SF16);
                    sum[0] = fmaf(s0, part[0], sum[0]);
                    sum[1] = fmaf(s0, part[1], sum[1]);
                    sum[2] = fmaf(s1, part[2], sum[2]);
                    sum[3] = fmaf(s1, part[3], sum[3]);
                };
                if constexpr (NT == 1) {  // x's fragments of the group stay, the tiles pass by
                    uint4 xp[GB][kParts];
#pragma unroll
                    for (int j = 0; j < GB; ++j) x_pairs(0, j, xp[j]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint32_t w0[GB], w1[GB];
                        words(m, 0, w0);
                        words(m, 1, w1);
                        const Zero<F16> z0(has_z ? zp[m * 16] & 15u : 8u), z1(has_z ? zp[m * 16 + 8] & 15u : 8u);
                        float part[4] = {};
#pragma unroll
                        for (int j = 0; j < GB; ++j) {
                            uint32_t lo[4], hi[4];
                            decode<F16>(w0[j], z0, lo);
                            decode<F16>(w1[j], z1, hi);
                            step(lo, hi, xp[j], part);
                        }
                        scale(m, part, acc[m][0]);
                    }
                } else {  // the tiles' codes stay decoded, x's tiles pass by
                    uint32_t w0[MT][GB], w1[MT][GB];
                    float part[MT][NT][4] = {};
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        words(m, 0, w0[m]);
                        words(m, 1, w1[m]);
                    }
#pragma unroll
                    for (int j = 0; j < GB; ++j) {
                        uint32_t lo[MT][4], hi[MT][4];
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            decode<F16>(w0[m][j], Zero<F16>(has_z ? zp[m * 16] & 15u : 8u), lo[m]);
                            decode<F16>(w1[m][j], Zero<F16>(has_z ? zp[m * 16 + 8] & 15u : 8u), hi[m]);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (8 * nt >= nr) break;
                            uint4 xp[kParts];
                            x_pairs(nt, j, xp);
#pragma unroll
                            for (int m = 0; m < MT; ++m) step(lo[m], hi[m], xp, part[m][nt]);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) scale(m, part[m][nt], acc[m][nt]);
                }
            }
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
        for (int i = tid; i < kTiles * 16 * nr; i += kWarps * 32) {
            const int ch = i & 15, m = i / 16 % kTiles, tok = i / (16 * kTiles);
            const int64_t n = n0 + 16 * m + ch;
            if (n >= N) continue;
            const int at = ((tok >> 3) * 32 + (ch & 7) * 4 + ((tok & 7) >> 1)) * 4 + (ch >> 3) * 2 + (tok & 1);
            const float *f = reinterpret_cast<const float *>(smem) + (ACT ? 2 * m : m) * NT * 128 + at;
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                v[0] += f[w * MT * NT * 128];
                if (ACT) v[1] += f[(w * MT + 1) * NT * 128];
            }
            st_act(a.y, (r0 + tok) * N + n, ACT ? swiglu_clamped(v[0], v[1], a.limit) : v[0], a.y_dtype);
        }
        __syncthreads();  // the buffers and s_x are used again
    }
}

// Launch with rows in tiles of 8 NT (2 where they are held).
template <int XD, int NT, int MT, int GB, bool ACT, bool SF16, bool HELD, int S>
int launch_tile(const Q4Args &a, cudaStream_t st) {
    using St = Stage<XD, NT, MT, GB, HELD>;
    constexpr int kTile = HELD ? 2 : 8 * NT;
    const int64_t most = a.rows < kTile ? a.rows : kTile;
    constexpr int sums = kWarps * MT * NT * 128 * (int)sizeof(float), kMost = kWarps * S * St::bytes(kTile);
    const int ring = kWarps * S * St::bytes((int)most);
    const int smem = ring > sums ? ring : sums;
    static_assert(kMost <= 226 * 1024 && kMost >= sums, "shared memory");
    auto kernel = matvec_kernel<XD, NT, MT, GB, ACT, SF16, HELD, S>;
    const int rc = set_smem_attr_once(reinterpret_cast<const void *>(kernel), kMost);
    if (rc) return rc;
    const int64_t tiles = cdiv(a.rows, kTile), per = cdiv(tiles, 65535);
    const dim3 grid((unsigned)cdiv(a.N, ACT ? 8 * MT : 16 * MT),
                    (unsigned)(a.offsets ? (a.E < a.rows ? a.E : a.rows) : cdiv(tiles, per)));
    VF_CUDA(launch_pdl(kernel, grid, dim3(kWarps * 32), (size_t)smem, st, a, (int)most, (int)per));
    VF_LAUNCH_CHECK("q4 matvec_kernel");
    return VFMOE_OK;
}

template <int XD, int GB, bool ACT, bool SF16>
int launch_rows(const Q4Args &a, cudaStream_t st) {
    // rows a tile: for sorted rows about twice the mean of the matrices that have some
    const int64_t mats = a.offsets ? (a.E < a.rows ? a.E : a.rows) : 1;
    const int64_t mean = cdiv(a.rows, mats);
    const int64_t want = a.offsets && a.rows > 8 ? 2 * mean : mean;
    constexpr bool F32 = XD == VFMOE_DT_F32;
    const int64_t tiles = a.N / 16 * (ACT ? 2 : 1) * mats;
    if (a.offsets ? a.rows * 4 <= a.E : a.rows <= 2) {
        if (tiles >= 4 * Q4B) return launch_tile<XD, 1, 4, GB, ACT, SF16, true, Q4S>(a, st);
        if constexpr (!ACT)
            if (tiles < 2 * 4 * 148) return launch_tile<XD, 1, 1, GB, false, SF16, true, 3>(a, st);
        return launch_tile<XD, 1, 2, GB, ACT, SF16, true, 3>(a, st);
    }
    if (want <= 8) {
        if (tiles >= 4 * Q4B) return launch_tile<XD, 1, 4, GB, ACT, SF16, false, 2>(a, st);
        return launch_tile<XD, 1, 2, GB, ACT, SF16, false, 3>(a, st);
    }
    if (want <= 16 || F32) return launch_tile<XD, 2, 2, GB, ACT, SF16, false, F32 ? 2 : 3>(a, st);
    return launch_tile<XD, F32 ? 2 : 4, 2, GB, ACT, SF16, false, 2>(a, st);
}

template <int XD, int GB>
int launch_group(const Q4Args &a, cudaStream_t st) {
    if (a.scale_f16) return a.up.data ? launch_rows<XD, GB, true, true>(a, st) : launch_rows<XD, GB, false, true>(a, st);
    return a.up.data ? launch_rows<XD, GB, true, false>(a, st) : launch_rows<XD, GB, false, false>(a, st);
}

template <int XD>
int launch_type(const Q4Args &a, cudaStream_t st) {
    return a.G == 32 ? launch_group<XD, 1>(a, st) : a.G == 64 ? launch_group<XD, 2>(a, st) : launch_group<XD, 4>(a, st);
}

}  // namespace q4
}  // namespace vfmoe
