// Products of 4-bit matrices with a few rows on the tensor cores (decode batches): y[r] = W x[r].
//
// W's codes are the m16n8k16 MMA's A operand, rows = output channels, and up to 8 NT rows of x its columns.  Per
// group of G elements the MMAs sum (q - z) x, both exact in the operand type (|q - z| <= 15; fp32 x goes as three bf16
// parts of 8 bits, each its own MMA), and the fp32 result is scaled once: y += s_g * part.
//
// What bounds it: W is read once, half a byte an element, so HBM should; but 8 codes of a bf16 operand take three shifts
// and four masks on the ALU pipe, which issues every other cycle, and at 6.4 TB/s that alone fills 60 % of it.  So a
// lane reads GB = G / 32 neighbouring words at a time, one set of scales serves GB steps, MT tiles of 16 channels share
// the x fragments, and mask and base go in one three-input operation.  N = 303,104, K = 6144, G = 128, one bf16 row:
// 208-216 us, 4.4-4.6 TB/s; without the decode 188, without the MMAs 208, without both 157.  Of what did not help: shifts as
// high products (+35 %), CTAs that keep their ring across tiles (+20 %: registers), 20 or 24 warps an SM instead of 16
// (+5, +10 %: more address arithmetic), two chains of sums a tile (+2 %), bf16 rows as scaled fp16 (fewer shifts, more else).
//
// A CTA owns 16 MT WM channels (half of that with gate and up: tiles alternate) and one tile of rows.  KW warps take K
// in chunks of 128 round robin, each streaming its own chunks of W, scales and x through its own shared-memory ring with
// cp.async, without a barrier among the warps; at the end the partial sums are added in warp order (the result does
// not depend on the launch) and the epilogue rounds once.  From 9 rows on x weighs more than W there, and WM warps of
// different channels share one ring of x instead, with a barrier a chunk.
//
// Any order of the elements within a step serves the product as long as both operands agree.  A word holds elements
// 8 w .. 8 w + 7; (word >> 4 i) & 0x000f000f is the pair (i, i + 4), so x's 8 elements are paired the same way.  Lane t of a
// quad takes the words t GB .. t GB + GB - 1 of a group, so all four lanes of an MMA lie in one group.
#pragma once

#include "common.cuh"
#include "q4.h"

namespace vfmoe {
namespace q4 {

constexpr int kSms = 148;
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

// Codes become operands by the known method of Kim, Henry, Fahim and Awadalla ("Who Says Elephants Can't Run", 2022): put into
// the low bits of a float whose step there is one, then subtract.
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

// Bytes of one warp's stage (W, scales, zero points) and of a row of x.  PAIRED rows are kept as MMA pairs, made once: one
// or two rows go through a lane's registers (HELD), rows that warps share are paired in place by the threads that copied
// them.  Else x stays as it lies in memory, and every use pairs it (a warp's own 8 rows cost the same either way).
template <int XD, bool PAIRED, int MT, int GB>
struct Stage {
    static constexpr int kGroups = 4 / GB;  // groups of a chunk
    static constexpr int kW = MT * 16 * 64;
    static constexpr int kS = kGroups * MT * 32;
    static constexpr int kZ = kGroups * MT * 16;
    static constexpr int kRow = XD != VFMOE_DT_F32 ? 256 : PAIRED ? 768 : 512;
    static constexpr int kOwn = kW + kS + kZ;
};

// KW warps share K; WM > 1 (with KW = 1): WM warps of other channels share the rows of x instead.
template <int XD, int NT, int MT, int GB, bool ACT, bool SF16, bool HELD, int KW, int WM, int S>
__global__ void __launch_bounds__(KW * WM * 32, (NT == 1 ? 16 : 12) / (KW * WM))
    matvec_kernel(Q4Args a, int x_rows_max, int row_tiles) {
    static_assert(WM == 1 || (KW == 1 && !HELD), "x is a warp's own, or the CTA's");
    constexpr int kWarps = KW, kThreads = KW * WM * 32;
    constexpr bool PAIRED = HELD || WM > 1;
    using St = Stage<XD, PAIRED, MT, GB>;
    constexpr int kTile = HELD ? 2 : 8 * NT;  // rows of x at a time
    constexpr bool F16 = XD == VFMOE_DT_F16, F32 = XD == VFMOE_DT_F32;
    constexpr int kParts = F32 ? 3 : 1;
    constexpr int es = F32 ? 4 : 2;
    constexpr int kTiles = ACT ? MT / 2 : MT;  // tiles of 16 channels of y
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_x[8 * NT];                     // byte offset of the tile's rows in x, -1: none
    __shared__ __align__(128) uint8_t s_zero[St::kRow];  // what lanes without a row read
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int wid = tid >> 5, warp = wid % KW, wm = wid / KW;  // place along K, and among the channels
    for (int i = tid * 4; i < St::kRow; i += kThreads * 4) *reinterpret_cast<uint32_t *>(s_zero + i) = 0u;

    // the matrix and its rows: blockIdx.y = a run of row tiles (one matrix), or the y-th matrix that has rows
    int64_t e = 0, row0 = 0, row1 = a.rows;
    if (a.offsets) {
        int left = blockIdx.y;
        e = -1;
        for (int b = 0; b < a.E && e < 0; b += 256) {
            int lo[8], hi[8];  // the offsets of 256 matrices in flight together
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = b + 32 * j + lane;
                lo[j] = i < a.E ? __ldg(a.offsets + i) : 0;
                hi[j] = i < a.E ? __ldg(a.offsets + i + 1) : 0;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned m = __ballot_sync(0xffffffffu, hi[j] > lo[j]);
                if (e < 0 && left < __popc(m)) {
                    for (; left > 0; --left) m &= m - 1;
                    const int src = __ffs(m) - 1;
                    e = b + 32 * j + src;
                    row0 = __shfl_sync(0xffffffffu, lo[j], src);
                    row1 = min((int64_t)__shfl_sync(0xffffffffu, hi[j], src), a.rows);
                }
                left -= __popc(m);
            }
        }
        if (e < 0 || row0 < 0) return;
    } else {
        row0 = blockIdx.y * (int64_t)kTile * row_tiles;
        row1 = min(row0 + (int64_t)kTile * row_tiles, a.rows);
    }

    const int64_t N = a.N, n0 = (blockIdx.x * (int64_t)WM + wm) * (16 * kTiles);
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

    // shared memory: per warp S stages of W, scales, zero points and (WM = 1) x; then the CTA's S stages of x
    const int x_bytes = x_rows_max * St::kRow, stage_bytes = St::kOwn + (WM == 1 ? x_bytes : 0);
    const int x_step = WM == 1 ? stage_bytes : x_bytes;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + wid * S * stage_bytes;
    uint8_t *const mine = smem + wid * S * stage_bytes;
    uint8_t *const x_ring = WM == 1 ? mine + St::kOwn : smem + WM * S * stage_bytes;
    const uint32_t w_dst = ring + wr * 64 + place_w<GB>(wr, wu) * 16;
    const uint32_t s_dst = ring + St::kW + sg * MT * 32 + sm * 32 + (lane & 1) * 16;
    const uint32_t z_dst = ring + St::kW + St::kS + zg * MT * 16 + zm * 16;
    static_assert(St::kGroups * MT * 2 <= 32, "one copy of scales a lane");

    for (int64_t r0 = row0; r0 < row1; r0 += kTile) {
        const int nr = (int)min((int64_t)kTile, row1 - r0);
        // W, scales and zero points of the warp's i-th chunk (chunk warp + i * kWarps of the row) into a stage
        auto fetch_w = [&](int i, int stage, int kv) {  // kv: elements left, a multiple of 32
            const uint32_t at = stage * stage_bytes;
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
        const int runs = (chunks - warp + kWarps - 1) / kWarps;  // chunks of this warp
        const int left0 = K - warp * kChunk;                     // elements from its first chunk on
        constexpr int kStep = kWarps * kChunk;
#pragma unroll
        for (int i = 0; i < S - 1; ++i)  // W does not wait for the row map
            if (i < runs) fetch_w(i, i, left0 - i * kStep);
        if (tid < 8 * NT) {
            const int64_t r = tid < nr ? (a.row_map ? a.row_map[r0 + tid] : r0 + tid) : -1;
            s_x[tid] = r >= 0 && r < a.x_rows ? r * K * es : -1;
        }
        __syncthreads();

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
        auto store_x = [&](int stage, int kv) {
            if (x_off >= 0 && xu * 8 < kv) {
                const int row = lane >> 4;
                uint8_t *dst = x_ring + stage * x_step + row * St::kRow + place_x<GB>(row, xu) * 16;
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
        // x, more rows: 16 lanes a row, kAtOnce rows at a time
        constexpr int kAtOnce = WM == 1 ? 2 : 2 * WM, kUnits = HELD ? 1 : 8 * NT / kAtOnce;
        const int x_row = WM == 1 ? lane >> 4 : tid >> 4;
        auto fetch_x = [&](int i, int stage, int kv) {
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(x_ring) + stage * x_step;
            if (xu * 8 < kv) {
#pragma unroll
                for (int j = 0; j < kUnits; ++j) {
                    if (kAtOnce * j >= nr) break;
                    const int row = kAtOnce * j + x_row;
                    const int64_t off = s_x[row];
                    if (off < 0) continue;
                    const uint8_t *src = x_src + off + (int64_t)i * (kWarps * kChunk * es);
                    const uint32_t dst = at + row * St::kRow + place_x<GB>(row, xu) * (8 * es);
                    cp16(dst, src);
                    if constexpr (F32) cp16(dst + 16, src + 16);
                }
            }
        };
        // the thread's own units of a stage that has arrived, paired (they need no barrier to be read; in fp32
        // the parts lie elsewhere, so all raw units are read first)
        auto pair_x = [&](int stage, int kv) {
            uint8_t *const base = x_ring + stage * x_step;
            uint4 raw[kUnits][F32 ? 2 : 1];
#pragma unroll
            for (int j = 0; j < kUnits; ++j) {
                const int row = kAtOnce * j + x_row;
                if (row >= nr || xu * 8 >= kv) continue;
                const uint4 *src = reinterpret_cast<const uint4 *>(base + row * St::kRow + place_x<GB>(row, xu) * (8 * es));
                raw[j][0] = src[0];
                if constexpr (F32) raw[j][1] = src[1];
            }
            if constexpr (F32) __syncthreads();
#pragma unroll
            for (int j = 0; j < kUnits; ++j) {
                const int row = kAtOnce * j + x_row;
                if (row >= nr || xu * 8 >= kv) continue;
                uint4 *dst = reinterpret_cast<uint4 *>(base + row * St::kRow + place_x<GB>(row, xu) * 16);
                if constexpr (F32) {
                    uint4 p[3];
                    pairs32(raw[j][0], raw[j][1], p);
#pragma unroll
                    for (int q = 0; q < 3; ++q) dst[16 * q] = p[q];
                } else {
                    dst[0] = pairs16(raw[j][0]);
                }
            }
        };

        float acc[MT][NT][4] = {};
        bool ok[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) ok[j] = 8 * j + g < kTile && s_x[8 * j + g] >= 0;

#pragma unroll
        for (int i = 0; i < S - 1; ++i) {
            if constexpr (!HELD)
                if (i < runs) fetch_x(i, i, left0 - i * kStep);
            cp_commit();
        }
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (i < runs) {
                    load_x(i, left0 - i * kStep);
                    store_x(i, left0 - i * kStep);
                }
            if (S - 1 < runs) load_x(S - 1, left0 - (S - 1) * kStep);
        }
        int stage = 0;
        for (int i = 0; i < runs; ++i) {
            cp_wait<S - 2>();
            // the stage is there for every lane (thread), and every one is done with the stage before it
            const int kv = left0 - i * kStep;
            if constexpr (WM == 1) {
                __syncwarp();
            } else {
                pair_x(stage, kv);
                __syncthreads();
            }
            if (i + S - 1 < runs) {
                const int into = stage == 0 ? S - 1 : stage - 1;
                const int kn = kv - (S - 1) * kStep;
                fetch_w(i + S - 1, into, kn);
                if constexpr (HELD) {
                    store_x(into, kn);
                    if (i + S < runs) load_x(i + S, kn - kStep);
                } else {
                    fetch_x(i + S - 1, into, kn);
                }
            }
            cp_commit();
            const uint8_t *buf = mine + stage * stage_bytes, *const xs = x_ring + stage * x_step;
            stage = stage == S - 1 ? 0 : stage + 1;
            const uint8_t *xb[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) xb[nt] = ok[nt] ? xs + (8 * nt + g) * St::kRow : s_zero;
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
                    if constexpr (PAIRED) {
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
#pragma unroll
                            for (int p = 0; p < kParts; ++p) {
                                mma<F16>(part, lo[0], hi[0], lo[1], hi[1], xp[j][p].x, xp[j][p].y);
                                mma<F16>(part, lo[2], hi[2], lo[3], hi[3], xp[j][p].z, xp[j][p].w);
                            }
                        }
                        scale(m, part, acc[m][0]);
                    }
                } else {  // the tiles' codes stay decoded, x's tiles pass by, two at a time: an MMA waits for the one
                          // before it on the same sums, so neighbours in program order do not share them
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
                        for (int nt = 0; nt < NT; nt += 2) {
                            if (8 * nt >= nr) break;
                            uint4 xp[2][kParts];
                            x_pairs(nt, j, xp[0]);
                            x_pairs(nt + 1, j, xp[1]);
#pragma unroll
                            for (int p = 0; p < kParts; ++p) {
#pragma unroll
                                for (int i = 0; i < 2 * MT; ++i) {
                                    const int m = i >> 1, q = i & 1;
                                    mma<F16>(part[m][nt + q], lo[m][0], hi[m][0], lo[m][1], hi[m][1], xp[q][p].x, xp[q][p].y);
                                }
#pragma unroll
                                for (int i = 0; i < 2 * MT; ++i) {
                                    const int m = i >> 1, q = i & 1;
                                    mma<F16>(part[m][nt + q], lo[m][2], hi[m][2], lo[m][3], hi[m][3], xp[q][p].z, xp[q][p].w);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) scale(m, part[m][nt], acc[m][nt]);
                }
            }
        }

        // the warps' sums, added in the order of K: [channels' warp][K's warp][tile][lane][4]
        cp_wait<0>();
        __syncthreads();
        float4 *red = reinterpret_cast<float4 *>(smem);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                red[((wid * MT + m) * NT + nt) * 32 + lane] =
                    make_float4(acc[m][nt][0], acc[m][nt][1], acc[m][nt][2], acc[m][nt][3]);
        __syncthreads();
        for (int i = tid; i < WM * kTiles * 16 * nr; i += kThreads) {
            const int ch = i & 15, m = i / 16 % kTiles, c = i / (16 * kTiles) % WM, tok = i / (16 * kTiles * WM);
            const int64_t n = (blockIdx.x * (int64_t)WM + c) * (16 * kTiles) + 16 * m + ch;
            if (n >= N) continue;
            const int at = ((tok >> 3) * 32 + (ch & 7) * 4 + ((tok & 7) >> 1)) * 4 + (ch >> 3) * 2 + (tok & 1);
            const float *f = reinterpret_cast<const float *>(smem) + (c * KW * MT + (ACT ? 2 * m : m)) * NT * 128 + at;
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                v[0] += f[w * MT * NT * 128];
                if (ACT) v[1] += f[(w * MT + 1) * NT * 128];
            }
            st_act(a.y, (r0 + tok) * N + n, ACT ? swiglu_clamped(v[0], v[1], a.limit) : v[0], a.y_dtype);
        }
        __syncthreads();  // the buffers and s_x are used again
    }
}

// Launch with rows in tiles of 8 NT (2 where they are held).
template <int XD, int NT, int MT, int GB, bool ACT, bool SF16, bool HELD, int KW, int WM, int S>
int launch_tile(const Q4Args &a, cudaStream_t st) {
    using St = Stage<XD, HELD || WM != 1, MT, GB>;
    constexpr int kTile = HELD ? 2 : 8 * NT;
    constexpr auto bytes = [](int rows) { return S * (KW * WM * St::kOwn + (WM == 1 ? KW : 1) * rows * St::kRow); };
    const int most = (int)(a.rows < kTile ? a.rows : kTile);
    constexpr int sums = KW * WM * MT * NT * 512, ring = bytes(kTile), top = ring > sums ? ring : sums;
    static_assert(top <= 224 * 1024, "shared memory");
    const int smem = bytes(most) > sums ? bytes(most) : sums;
    auto kernel = matvec_kernel<XD, NT, MT, GB, ACT, SF16, HELD, KW, WM, S>;
    const int rc = set_smem_attr_once(reinterpret_cast<const void *>(kernel), top);
    if (rc) return rc;
    const int64_t tiles = cdiv(a.rows, kTile), per = cdiv(tiles, 65535);
    const dim3 grid((unsigned)cdiv(a.N, (ACT ? 8 : 16) * MT * WM),
                    (unsigned)(a.offsets ? (a.E < a.rows ? a.E : a.rows) : cdiv(tiles, per)));
    VF_CUDA(launch_pdl(kernel, grid, dim3(KW * WM * 32), (size_t)smem, st, a, most, (int)per));
    VF_LAUNCH_CHECK("q4 matvec_kernel");
    return VFMOE_OK;
}

// One tile of rows: channels a CTA and warps along K by what there is to spread (`tiles`: MMA tiles of 16 channels over all
// matrices).  Up to two CTAs an SM take 8 warps each, up to 4 a single tile (two with gate and up), from there on wide tiles:
//   N = 6144, K = 6144, one row (384 tiles): 8 warps 13.2 us, 4 warps 11.0;  N = 2048 (128): 8.1, 8.4
//   8 matrices of N = 6144, K = 2048 (3,072 tiles): 64 channels 19.7 us, 32 channels 21.5
template <int XD, int GB, bool ACT, bool SF16, bool HELD>
int launch_few(const Q4Args &a, int64_t tiles, cudaStream_t st) {
    constexpr int A = ACT ? 2 : 1;
    if (tiles <= 2 * A * kSms) return launch_tile<XD, 1, A, GB, ACT, SF16, HELD, 8, 1, 2>(a, st);
    if (tiles <= 4 * A * kSms) return launch_tile<XD, 1, A, GB, ACT, SF16, HELD, 4, 1, 3>(a, st);
    if (!ACT && tiles <= 8 * kSms) return launch_tile<XD, 1, 2, GB, ACT, SF16, HELD, 4, 1, 3>(a, st);
    return launch_tile<XD, 1, 4, GB, ACT, SF16, HELD, 4, 1, 2>(a, st);
}

// Rows a tile: all of a dense call; for sorted rows about twice the mean of the matrices that have some.  One or two rows (sorted:
// at most one for four matrices) are held in registers on their way and paired once; a matrix with more rows than its
// tile takes them in turns.
// More than 8 rows: shared x where that leaves enough CTAs, else warps along K:
//   n = 16, N = 2048, K = 6144: along K 9.6 us (fp16), 64 CTAs of 32 channels 18.9
//   n = 32, N = 131072, K = 6144: shared 265 us, along K 430;  n = 256, N = 6144: shared 115 us, along K 204
//   n = 32, N = 2048, K = 6144: along K 20 us, shared 66;  n = 64, N = 6144, K = 2048: along K 24.5, shared 29
// fp32 rows of more than 16 a tile always share x.  Along K they fit too (150 KB of shared memory), with a border of their own:
//   n = 32, N = 2048, K = 6144: along K 48 us, shared 131;  N = 6144: 133, 139;  n = 24, N = 12288, K = 2048: 63, 47;
//   n = 64, N = 6144, K = 2048: 95, 47
template <int XD, int GB, bool ACT, bool SF16>
int launch_rows(const Q4Args &a, cudaStream_t st) {
    constexpr int A = ACT ? 2 : 1;
    constexpr bool F32 = XD == VFMOE_DT_F32;
    const int64_t mats = a.offsets ? (a.E < a.rows ? a.E : a.rows) : 1;
    const int64_t mean = cdiv(a.rows, mats);
    const int64_t want = a.offsets && a.rows > 8 ? 2 * mean : mean;
    const int64_t tiles = a.N / 16 * A * mats;
    if (a.offsets ? a.rows * 4 <= a.E : a.rows <= 2) return launch_few<XD, GB, ACT, SF16, true>(a, tiles, st);
    if (want <= 8) return launch_few<XD, GB, ACT, SF16, false>(a, tiles, st);
    if (want <= 16) {
        if (tiles < 4 * A * kSms) return launch_tile<XD, 2, A, GB, ACT, SF16, false, 8, 1, 2>(a, st);
        return launch_tile<XD, 2, 2, GB, ACT, SF16, false, 1, 4, 3>(a, st);
    }
    const int64_t all = tiles * (a.offsets ? 1 : cdiv(a.rows, 32));
    if constexpr (!F32)
        if (all < 6 * A * kSms) return launch_tile<XD, 4, A, GB, ACT, SF16, false, 4, 1, 2>(a, st);
    return launch_tile<XD, 4, 2, GB, ACT, SF16, false, 1, 4, 3>(a, st);
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
