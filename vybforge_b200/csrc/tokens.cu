// Tokens sorted by expert and back, in the caller's own element type, with their gradients.
//
//   permute           pos_of[t,l] = rank of lane (t, l) among the kept lanes ordered by (expert, token, lane)
//                     xs[pos_of[t,l]] = x[t]
//   permute backward  dx[t] = sum_l dxs[pos_of[t,l]]
//   combine           out[t] = sum_l w[t,l] y[pos_of[t,l]] (+ y_shared[t])
//   combine backward  dy[pos_of[t,l]] = w[t,l] dout[t],  dw[t,l] = <dout[t], y[pos_of[t,l]]>
//
// A lane is kept when its id lies in [0, E); the others have position -1 and no row.  All four move
// every row once and compute next to nothing, so HBM bandwidth bounds them at prefill sizes and launch
// latency at decode sizes: one CTA works on one token, its k row positions in shared memory, and reads
// or writes the token's row once for all of its lanes.  Sums run in fp32 in lane order (one thread owns
// a column) with one rounding at the end, so results do not depend on the launch.
#include "common.cuh"
#include "kernels.h"

namespace vfmoe {

namespace {

// ----------------------------------------------------------------------------- vectors of VE elements
template <int DT> struct Elem;
template <> struct Elem<VFMOE_DT_F32> { using type = float; };
template <> struct Elem<VFMOE_DT_F16> { using type = __half; };
template <> struct Elem<VFMOE_DT_BF16> { using type = __nv_bfloat16; };

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::type v) {
    if constexpr (DT == VFMOE_DT_F32) return v;
    else if constexpr (DT == VFMOE_DT_F16) return __half2float(v);
    else return __bfloat162float(v);
}

template <int DT>
__device__ __forceinline__ typename Elem<DT>::type from_f32(float v) {
    if constexpr (DT == VFMOE_DT_F32) return v;
    else if constexpr (DT == VFMOE_DT_F16) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

// VE elements as they lie in memory: one or two 16-byte words, one 8-byte word, or one element.
template <int DT, int VE>
struct alignas(sizeof(typename Elem<DT>::type) * VE >= 16 ? 16 : sizeof(typename Elem<DT>::type) * VE) Vec {
    typename Elem<DT>::type e[VE];
};

template <int DT, int VE>
__device__ __forceinline__ Vec<DT, VE> ldv(const void *p, int64_t i) {
    return *reinterpret_cast<const Vec<DT, VE> *>(reinterpret_cast<const typename Elem<DT>::type *>(p) + i);
}

template <int DT, int VE>
__device__ __forceinline__ void stv(void *p, int64_t i, const float (&v)[VE]) {
    Vec<DT, VE> o;
#pragma unroll
    for (int j = 0; j < VE; ++j) o.e[j] = from_f32<DT>(v[j]);
    *reinterpret_cast<Vec<DT, VE> *>(reinterpret_cast<typename Elem<DT>::type *>(p) + i) = o;
}

template <int VE>
__device__ __forceinline__ void stv_dt(void *p, int64_t i, const float (&v)[VE], int dtype) {
    if (dtype == VFMOE_DT_BF16) stv<VFMOE_DT_BF16, VE>(p, i, v);
    else if (dtype == VFMOE_DT_F16) stv<VFMOE_DT_F16, VE>(p, i, v);
    else stv<VFMOE_DT_F32, VE>(p, i, v);
}

template <int DT, int VE>
__device__ __forceinline__ void ldv_f32(const void *p, int64_t i, float (&v)[VE]) {
    const Vec<DT, VE> u = ldv<DT, VE>(p, i);
#pragma unroll
    for (int j = 0; j < VE; ++j) v[j] = to_f32<DT>(u.e[j]);
}

template <int VE>
__device__ __forceinline__ void ldv_dt(const void *p, int64_t i, float (&v)[VE], int dtype) {
    if (dtype == VFMOE_DT_BF16) ldv_f32<VFMOE_DT_BF16, VE>(p, i, v);
    else if (dtype == VFMOE_DT_F16) ldv_f32<VFMOE_DT_F16, VE>(p, i, v);
    else ldv_f32<VFMOE_DT_F32, VE>(p, i, v);
}

inline int elem_size(int dtype) { return dtype == VFMOE_DT_F32 ? 4 : 2; }

// threads of a CTA that walks n vectors: whole warps, 256 at most
inline unsigned row_threads(int64_t n) { return n >= 256 ? 256u : (unsigned)(cdiv(n, 32) * 32); }

// ----------------------------------------------------------------------------- plan
constexpr int kPlanLanes = 1024;   // lanes of one chunk (one thread each)
constexpr int kSmallLanes = 2048;  // up to here every CTA ranks its own token's lanes by itself

__device__ __forceinline__ bool kept_id(int e, int E) { return e >= 0 && e < E; }

// x[t] to its k rows; pos: the token's row positions in shared memory (-1: none).
template <typename V>
__device__ __forceinline__ void copy_rows(const void *x, void *xs, int64_t t, int64_t nv, const int *pos, int k) {
    const V *src = reinterpret_cast<const V *>(x) + t * nv;
    V *dst = reinterpret_cast<V *>(xs);
    for (int64_t c = threadIdx.x; c < nv; c += blockDim.x) {
        const V v = src[c];
        for (int l = 0; l < k; ++l) {
            const int p = pos[l];
            if (p >= 0) dst[(int64_t)p * nv + c] = v;
        }
    }
}

// Exclusive scan over the CTA (blockDim.x a multiple of 32, at most 1024) of one value a thread;
// *total gets the sum.
__device__ __forceinline__ int block_exclusive(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < nw; ++w) {
        before += w < warp ? warp_sums[w] : 0;
        all += warp_sums[w];
    }
    __syncthreads();
    *total = all;
    return before + inc - v;
}

// One launch for up to kSmallLanes lanes (a decode batch).  The ids of all lanes fit in shared memory,
// so CTA t ranks its own k lanes by counting (one warp a lane): kept ids below, and equal ids earlier.
// CTA T writes counts, offsets and the -1 tail of perm_tok.
template <typename V>
__global__ void __launch_bounds__(256) permute_small_kernel(const int32_t *__restrict__ idx, int T, int k, int E,
                                                            const void *__restrict__ x, void *__restrict__ xs,
                                                            int64_t nv, int32_t *__restrict__ counts,
                                                            int32_t *__restrict__ offsets,
                                                            int32_t *__restrict__ perm_tok,
                                                            int32_t *__restrict__ pos_of) {
    __shared__ int s_id[kSmallLanes];
    __shared__ int s_hist[1024];
    __shared__ int s_pos[32];
    __shared__ int s_ws[32];
    const int n = T * k, t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    for (int i = threadIdx.x; i < n; i += blockDim.x) s_id[i] = idx[i];
    if (t == T) {
        for (int e = threadIdx.x; e < E; e += blockDim.x) s_hist[e] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x)
            if (kept_id(s_id[i], E)) atomicAdd(&s_hist[s_id[i]], 1);
        __syncthreads();
        const int per = (E + blockDim.x - 1) / blockDim.x;
        int mine = 0;
        for (int i = 0; i < per; ++i) {
            const int e = threadIdx.x * per + i;
            mine += e < E ? s_hist[e] : 0;
        }
        int total;
        int at = block_exclusive(mine, s_ws, &total);
        for (int i = 0; i < per; ++i) {
            const int e = threadIdx.x * per + i;
            if (e >= E) break;
            counts[e] = s_hist[e];
            offsets[e] = at;
            at += s_hist[e];
        }
        if (threadIdx.x == 0) offsets[E] = total;
        for (int i = total + threadIdx.x; i < n; i += blockDim.x) perm_tok[i] = -1;
        return;
    }
    __syncthreads();
    for (int l = warp; l < k; l += nw) {
        const int me = t * k + l, e = s_id[me];
        int r = 0;
        for (int i = lane; i < n; i += 32) {
            const int o = s_id[i];
            r += (o >= 0 && (o < e || (o == e && i < me))) ? 1 : 0;
        }
        r = __reduce_add_sync(0xffffffffu, r);
        if (lane == 0) {
            const int p = kept_id(e, E) ? r : -1;
            s_pos[l] = p;
            pos_of[me] = p;
            if (p >= 0) perm_tok[p] = t;
        }
    }
    __syncthreads();
    if (x) copy_rows<V>(x, xs, t, nv, s_pos, k);
}

// Larger batches, first of three launches: one CTA ranks the lanes of one chunk among themselves.  Lanes of
// a warp with the same id find each other with a match; the warps' counts of an expert are summed in warp
// order, so the order is that of the lanes.  Writes the rank within the chunk (to pos_of) and hist[chunk][e].
__global__ void __launch_bounds__(kPlanLanes) plan_chunk_kernel(const int32_t *__restrict__ idx, int64_t n, int E,
                                                                int32_t *__restrict__ hist,
                                                                int32_t *__restrict__ pos_of) {
    extern __shared__ uint16_t s_cnt[];  // [32 warps][E]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = blockIdx.x * (int64_t)kPlanLanes + threadIdx.x;
    const int id = i < n ? idx[i] : -1;
    const bool kept = kept_id(id, E);
    for (int j = threadIdx.x; j < 32 * E; j += kPlanLanes) s_cnt[j] = 0;
    __syncthreads();
    const unsigned same = __match_any_sync(0xffffffffu, kept ? id : -1);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (kept && before == 0) s_cnt[warp * E + id] = (uint16_t)__popc(same);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kPlanLanes) {
        int sum = 0;
#pragma unroll 8
        for (int w = 0; w < 32; ++w) {
            const int c = s_cnt[w * E + e];
            s_cnt[w * E + e] = (uint16_t)sum;
            sum += c;
        }
        hist[blockIdx.x * (int64_t)E + e] = sum;
    }
    __syncthreads();
    if (i < n) pos_of[i] = kept ? s_cnt[warp * E + id] + before : -1;
}

// Second launch, one CTA: hist[chunk][e] becomes the first row of expert e's lanes of that chunk.  The
// threads form groups of Ep (E rounded up to whole warps); each group sums a run of chunks of every expert.
__global__ void __launch_bounds__(1024) plan_scan_kernel(int32_t *__restrict__ hist, int C, int E, int64_t n,
                                                         int32_t *__restrict__ counts, int32_t *__restrict__ offsets,
                                                         int32_t *__restrict__ perm_tok) {
    __shared__ int s_part[1024];
    __shared__ int s_ws[32];
    pdl_wait_then_release();
    const int Ep = (E + 31) / 32 * 32, groups = 1024 / Ep;
    const int g = threadIdx.x / Ep, e = threadIdx.x % Ep;
    const int run = (C + groups - 1) / groups;
    const bool work = g < groups && e < E;
    const int c0 = min(C, g * run), c1 = min(C, c0 + run);
    int sum = 0;
    if (work) {
#pragma unroll 8
        for (int c = c0; c < c1; ++c) sum += hist[(int64_t)c * E + e];
    }
    s_part[threadIdx.x] = sum;
    __syncthreads();
    int tot = 0, before = 0;
    if (work)
        for (int j = 0; j < groups; ++j) {
            const int v = s_part[j * Ep + e];
            before += j < g ? v : 0;
            tot += v;
        }
    int total;
    const int off = block_exclusive(g == 0 && work ? tot : 0, s_ws, &total);
    __syncthreads();
    if (g == 0 && work) {
        counts[e] = tot;
        offsets[e] = off;
        s_part[e] = off;
    }
    if (threadIdx.x == 0) offsets[E] = total;
    __syncthreads();
    if (work) {
        int at = s_part[e] + before;
#pragma unroll 8
        for (int c = c0; c < c1; ++c) {
            const int v = hist[(int64_t)c * E + e];
            hist[(int64_t)c * E + e] = at;
            at += v;
        }
    }
    for (int64_t i = total + threadIdx.x; i < n; i += 1024) perm_tok[i] = -1;
}

// Third launch, one CTA a token: final positions, and the token's row to each of them.
template <typename V>
__global__ void __launch_bounds__(256) permute_rows_kernel(const int32_t *__restrict__ idx, int k, int E,
                                                           const int32_t *__restrict__ base,
                                                           const void *__restrict__ x, void *__restrict__ xs,
                                                           int64_t nv, int32_t *__restrict__ perm_tok,
                                                           int32_t *__restrict__ pos_of) {
    __shared__ int s_pos[32];
    pdl_wait_then_release();
    const int64_t t = blockIdx.x;
    if (threadIdx.x < k) {
        const int64_t i = t * k + threadIdx.x;
        const int e = idx[i];
        int p = -1;
        if (kept_id(e, E)) {
            p = base[i / kPlanLanes * E + e] + pos_of[i];
            pos_of[i] = p;
            perm_tok[p] = (int)t;
        }
        s_pos[threadIdx.x] = p;
    }
    __syncthreads();
    if (x) copy_rows<V>(x, xs, t, nv, s_pos, k);
}

template <typename V>
int permute_launch(const int32_t *idx, int64_t T, int k, int E, const void *x, void *xs, int64_t nv, int32_t *counts,
                   int32_t *offsets, int32_t *perm_tok, int32_t *pos_of, int32_t *ws, cudaStream_t st) {
    const int64_t n = T * k;
    const unsigned th = x ? row_threads(nv) : 256u;
    if (n <= kSmallLanes) {
        permute_small_kernel<V><<<(unsigned)T + 1, 256, 0, st>>>(idx, (int)T, k, E, x, xs, nv, counts, offsets,
                                                                 perm_tok, pos_of);
        VF_LAUNCH_CHECK("permute_small_kernel");
        return VFMOE_OK;
    }
    const int64_t C = cdiv(n, kPlanLanes);
    const int smem = 32 * E * (int)sizeof(uint16_t);
    if (smem > 48 * 1024) {
        const int rc = set_smem_attr_once(reinterpret_cast<const void *>(plan_chunk_kernel), smem);
        if (rc) return rc;
    }
    plan_chunk_kernel<<<(unsigned)C, kPlanLanes, smem, st>>>(idx, n, E, ws, pos_of);
    VF_LAUNCH_CHECK("plan_chunk_kernel");
    VF_CUDA(launch_pdl(plan_scan_kernel, dim3(1), dim3(1024), 0, st, ws, (int)C, E, n, counts, offsets, perm_tok));
    VF_LAUNCH_CHECK("plan_scan_kernel");
    VF_CUDA(launch_pdl(permute_rows_kernel<V>, dim3((unsigned)T), dim3(th), 0, st, idx, k, E, ws, x, xs, nv, perm_tok,
                       pos_of));
    VF_LAUNCH_CHECK("permute_rows_kernel");
    return VFMOE_OK;
}

// ----------------------------------------------------------------------------- way back
// out[t] = sum_l w[t,l] y[pos_of[t,l]] (+ y_shared[t]); one thread owns VE columns and adds the lanes in
// order, their loads independent of each other.
template <int DT, int VE>
__global__ void __launch_bounds__(256) return_rows_kernel(const void *__restrict__ y, const int32_t *__restrict__ pos_of,
                                                          const float *__restrict__ w, int64_t H, int k,
                                                          const void *__restrict__ y_shared, void *__restrict__ out,
                                                          int out_dtype) {
    __shared__ int64_t s_at[32];
    __shared__ float s_w[32];
    const int64_t t = blockIdx.x;
    if (threadIdx.x < k) {
        const int32_t p = pos_of[t * k + threadIdx.x];
        s_at[threadIdx.x] = p < 0 ? -1 : (int64_t)p * H;
        s_w[threadIdx.x] = w ? w[t * k + threadIdx.x] : 1.0f;
    }
    __syncthreads();
    for (int64_t c = (blockIdx.y * (int64_t)blockDim.x + threadIdx.x) * VE; c < H;
         c += (int64_t)gridDim.y * blockDim.x * VE) {
        float acc[VE] = {};
#pragma unroll 8
        for (int l = 0; l < k; ++l) {
            if (s_at[l] < 0) continue;
            const Vec<DT, VE> v = ldv<DT, VE>(y, s_at[l] + c);
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] = fmaf(s_w[l], to_f32<DT>(v.e[j]), acc[j]);
        }
        if (y_shared) {
            const Vec<DT, VE> v = ldv<DT, VE>(y_shared, t * H + c);
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += to_f32<DT>(v.e[j]);
        }
        stv_dt<VE>(out, t * H + c, acc, out_dtype);
    }
}

// dy[pos] = w dout[t] and dw = <dout[t], y[pos]>, one CTA a token, lanes in groups of 8: a thread loads its
// columns of dout once a group and the 8 rows' columns together, before it writes them (so dy may be y).
template <int DT, int VE>
__global__ void __launch_bounds__(256) combine_backward_kernel(const void *dout, int dout_dtype, const void *y,
                                                               const int32_t *__restrict__ pos_of,
                                                               const float *__restrict__ w, int64_t H, int k, void *dy,
                                                               float *__restrict__ dw) {
    __shared__ int64_t s_at[32];
    __shared__ float s_w[32];
    __shared__ float s_dot[8][8];
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if (threadIdx.x < k) {
        const int32_t p = pos_of[t * k + threadIdx.x];
        s_at[threadIdx.x] = p < 0 ? -1 : (int64_t)p * H;
        s_w[threadIdx.x] = w ? w[t * k + threadIdx.x] : 1.0f;
    }
    __syncthreads();
    for (int l0 = 0; l0 < k; l0 += 8) {
        float dot[8] = {};
        for (int64_t c = (int64_t)threadIdx.x * VE; c < H; c += (int64_t)blockDim.x * VE) {
            float d[VE];
            ldv_dt<VE>(dout, t * H + c, d, dout_dtype);
            Vec<DT, VE> v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (dw && l0 + i < k && s_at[l0 + i] >= 0) v[i] = ldv<DT, VE>(y, s_at[l0 + i] + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (l0 + i >= k || s_at[l0 + i] < 0) continue;
                if (dw) {
#pragma unroll
                    for (int j = 0; j < VE; ++j) dot[i] = fmaf(d[j], to_f32<DT>(v[i].e[j]), dot[i]);
                }
                if (dy) {
                    float o[VE];
#pragma unroll
                    for (int j = 0; j < VE; ++j) o[j] = s_w[l0 + i] * d[j];
                    stv<DT, VE>(dy, s_at[l0 + i] + c, o);
                }
            }
        }
        if (!dw) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = warp_sum_f32(dot[i]);
            if (lane == 0) s_dot[warp][i] = s;
        }
        __syncthreads();
        if (threadIdx.x < 8 && l0 + threadIdx.x < k) {
            float s = 0.f;
            for (int u = 0; u < nw; ++u) s += s_dot[u][threadIdx.x];
            dw[t * k + l0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
}

template <int DT, int VE>
int return_launch(const void *y, const int32_t *pos_of, const float *w, int64_t T, int64_t H, int k,
                  const void *y_shared, void *out, int out_dtype, cudaStream_t st) {
    const unsigned th = row_threads(H / VE);
    const int64_t cols = cdiv(H / VE, th);
    const dim3 grid((unsigned)T, (unsigned)(cols < 65535 ? cols : 65535));
    return_rows_kernel<DT, VE><<<grid, th, 0, st>>>(y, pos_of, w, H, k, y_shared, out, out_dtype);
    VF_LAUNCH_CHECK("return_rows_kernel");
    return VFMOE_OK;
}

template <int DT, int VE>
int combine_backward_launch(const void *dout, int dout_dtype, const void *y, const int32_t *pos_of, const float *w,
                            int64_t T, int64_t H, int k, void *dy, float *dw, cudaStream_t st) {
    combine_backward_kernel<DT, VE><<<(unsigned)T, row_threads(H / VE), 0, st>>>(dout, dout_dtype, y, pos_of, w, H, k,
                                                                               dy, dw);
    VF_LAUNCH_CHECK("combine_backward_kernel");
    return VFMOE_OK;
}

inline bool aligned(const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

int64_t permute_ws_bytes(int64_t T, int k, int E) {
    const int64_t n = T * k;
    return n <= kSmallLanes ? 0 : cdiv(n, kPlanLanes) * E * (int64_t)sizeof(int32_t);
}

// Rows move as 16-byte words where their length and both addresses allow, else element by element.
int launch_permute(const int32_t *idx, int64_t T, int k, int E, const void *x, int dtype, int64_t H, void *xs,
                   int32_t *counts, int32_t *offsets, int32_t *perm_tok, int32_t *pos_of, int32_t *ws,
                   cudaStream_t st) {
    const int64_t bytes = H * elem_size(dtype);
    if (bytes % 16 == 0 && aligned(x, 16) && aligned(xs, 16))
        return permute_launch<uint4>(idx, T, k, E, x, xs, bytes / 16, counts, offsets, perm_tok, pos_of, ws, st);
    if (elem_size(dtype) == 4)
        return permute_launch<uint32_t>(idx, T, k, E, x, xs, H, counts, offsets, perm_tok, pos_of, ws, st);
    return permute_launch<uint16_t>(idx, T, k, E, x, xs, H, counts, offsets, perm_tok, pos_of, ws, st);
}

// 16-byte words of y (8 columns of a 16-bit type, 4 of fp32) where rows and addresses allow, else columns.
int launch_return_rows(const void *y, int y_dtype, const int32_t *pos_of, const float *w, int64_t T, int64_t H, int k,
                       const void *y_shared, void *out, int out_dtype, cudaStream_t st) {
    const int ve = 16 / elem_size(y_dtype);
    const int64_t oa = ve * elem_size(out_dtype) < 16 ? ve * elem_size(out_dtype) : 16;
    const bool wide = H % ve == 0 && aligned(y, 16) && aligned(y_shared, 16) && aligned(out, oa);
#define VF_RETURN(DT, VE) return return_launch<DT, VE>(y, pos_of, w, T, H, k, y_shared, out, out_dtype, st)
    if (y_dtype == VFMOE_DT_F32) {
        if (wide) VF_RETURN(VFMOE_DT_F32, 4);
        VF_RETURN(VFMOE_DT_F32, 1);
    }
    if (y_dtype == VFMOE_DT_F16) {
        if (wide) VF_RETURN(VFMOE_DT_F16, 8);
        VF_RETURN(VFMOE_DT_F16, 1);
    }
    if (wide) VF_RETURN(VFMOE_DT_BF16, 8);
    VF_RETURN(VFMOE_DT_BF16, 1);
#undef VF_RETURN
}

int launch_combine_backward(const void *dout, int dout_dtype, const void *y, int y_dtype, const int32_t *pos_of,
                            const float *w, int64_t T, int64_t H, int k, void *dy, float *dw, cudaStream_t st) {
    const int ve = 16 / elem_size(y_dtype);
    const bool wide = H % ve == 0 && aligned(y, 16) && aligned(dy, 16) && aligned(dout, 16);
#define VF_BACK(DT, VE) return combine_backward_launch<DT, VE>(dout, dout_dtype, y, pos_of, w, T, H, k, dy, dw, st)
    if (y_dtype == VFMOE_DT_F32) {
        if (wide) VF_BACK(VFMOE_DT_F32, 4);
        VF_BACK(VFMOE_DT_F32, 1);
    }
    if (y_dtype == VFMOE_DT_F16) {
        if (wide) VF_BACK(VFMOE_DT_F16, 8);
        VF_BACK(VFMOE_DT_F16, 1);
    }
    if (wide) VF_BACK(VFMOE_DT_BF16, 8);
    VF_BACK(VFMOE_DT_BF16, 1);
#undef VF_BACK
}

}  // namespace vfmoe
