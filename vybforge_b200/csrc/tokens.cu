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
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"
#include "kernels.h"

namespace vfmoe {

namespace cg = cooperative_groups;

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
constexpr int kPlanCtas = 8;       // CTAs of the plan's cluster
constexpr int kPlanBatch = 8;      // ids a lane holds at a time
// Up to here every CTA ranks its own token's lanes by itself, in the one launch that copies the rows: 3.9 us at
// 256 lanes and 8.9 at 2,048, where the cluster's plan and the copy take 13.2 (E = 256, cold caches).
constexpr int kSmallLanes = 2048;

__device__ __forceinline__ bool kept_id(int e, int E) { return e >= 0 && e < E; }

// A token's row to its k rows.  load() fetches the thread's first kHeld words before the positions are
// known; store() writes them and moves the rest; pos: the row positions in shared memory (-1: none).
template <typename V>
struct RowCopy {
    static constexpr int kHeld = 4;
    V v[kHeld];
    __device__ __forceinline__ void load(const void *x, int64_t t, int64_t nv) {
        const V *src = reinterpret_cast<const V *>(x) + t * nv;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int64_t c = threadIdx.x + j * (int64_t)blockDim.x;
            if (c < nv) v[j] = src[c];
        }
    }
    __device__ __forceinline__ void store(const void *x, void *xs, int64_t t, int64_t nv, const int *pos, int k) {
        const V *src = reinterpret_cast<const V *>(x) + t * nv;
        V *dst = reinterpret_cast<V *>(xs);
        for (int l = 0; l < k; ++l) {
            const int p = pos[l];
            if (p < 0) continue;
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int64_t c = threadIdx.x + j * (int64_t)blockDim.x;
                if (c < nv) dst[(int64_t)p * nv + c] = v[j];
            }
        }
        for (int64_t c = threadIdx.x + kHeld * (int64_t)blockDim.x; c < nv; c += blockDim.x) {
            const V u = src[c];
            for (int l = 0; l < k; ++l) {
                const int p = pos[l];
                if (p >= 0) dst[(int64_t)p * nv + c] = u;
            }
        }
    }
};

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
    // every warp scans the warps' sums for itself
    const int mine = lane < nw ? warp_sums[lane] : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    const int before = __shfl_sync(0xffffffffu, sum - mine, warp);
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
    pdl_wait_then_release();
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
    RowCopy<V> row;
    if (x) row.load(x, t, nv);
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
    if (x) row.store(x, xs, t, nv, s_pos, k);
}

// lanes of the warp with this lane's id (its low `bits` bits, and whether it is negative)
__device__ __forceinline__ unsigned same_id(int id, int bits) {
    const unsigned none = __ballot_sync(0xffffffffu, id < 0);
    unsigned m = id < 0 ? none : ~none;
    for (int b = 0; b < bits; ++b) {
        const unsigned set = __ballot_sync(0xffffffffu, (id >> b) & 1);
        m &= (id >> b) & 1 ? set : ~set;
    }
    return m;
}

// the next kPlanBatch ids of a lane, -1 for a dropped one or none; their loads in flight together
__device__ __forceinline__ void load_ids(const int32_t *__restrict__ idx, int64_t i, int64_t end, int E,
                                         int (&id)[kPlanBatch]) {
#pragma unroll
    for (int j = 0; j < kPlanBatch; ++j) id[j] = i + 32 * j < end ? idx[i + 32 * j] : -1;
#pragma unroll
    for (int j = 0; j < kPlanBatch; ++j)
        if (!kept_id(id[j], E)) id[j] = -1;
}

// Larger batches: the plan in one launch of one cluster.  Each of its warps owns a run of lanes.  The ids
// are read twice: first every warp counts its lanes of each expert in shared memory; the counts are summed
// over the warps of a CTA, over the CTAs (distributed shared memory) and over the experts, which leaves in
// each warp's counter the first row of its lanes of that expert; then the warp hands out rows 32 lanes at a
// time, lanes with the same id finding each other by one ballot a bit of the id.  Runs and lanes ascend, so the order is
// that of the lanes.  65,536 lanes, E = 256: 10.9 us with cold caches, 9.8 at 32,768, 8 of them the launch and
// the chain of loads, barriers and sums.  (Three grid-wide launches, chunk ranks, a scan and the positions,
// took 21 us; a match instead of the ballots 4 us more; writing perm_tok here as well, 32 scattered sectors a
// store from 8 SMs, 4 us more, so the next kernel does it.)
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(1024)
    plan_kernel(const int32_t *__restrict__ idx, int64_t n, int k, int E, int32_t *__restrict__ counts,
                int32_t *__restrict__ offsets, int32_t *__restrict__ perm_tok, int32_t *__restrict__ pos_of) {
    extern __shared__ int s_cnt[];  // [32 warps][E]
    __shared__ int s_tot[1024];
    __shared__ int s_ws[32];
    // launched after its predecessor's end: the rows kernel may be set up, and load x, meanwhile
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
    const int64_t run = (n + kPlanCtas * 1024 - 1) / (kPlanCtas * 1024) * 32;
    const int64_t i0 = (rank * 32 + warp) * run + lane, i1 = min(n, (int64_t)(rank * 32 + warp + 1) * run);
    int *cnt = s_cnt + warp * E;
    const int bits = 32 - __clz(E - 1);  // 0 for E = 1
    int id[kPlanBatch];
    load_ids(idx, i0, i1, E, id);
    for (int j = threadIdx.x; j < 32 * E; j += 1024) s_cnt[j] = 0;
    __syncthreads();
    for (int64_t i = i0; i - lane < i1; i += 32 * kPlanBatch) {
        if (i != i0) load_ids(idx, i, i1, E, id);
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j)
            if (id[j] >= 0) atomicAdd(&cnt[id[j]], 1);
    }
    __syncthreads();
    int c[32], mine = 0;  // the warps' counts of expert e
    if (e < E) {
#pragma unroll
        for (int w = 0; w < 32; ++w) c[w] = s_cnt[w * E + e];
#pragma unroll
        for (int w = 0; w < 32; ++w) mine += c[w];
    }
    s_tot[e] = mine;
    cl.sync();
    int before = 0, all = 0;
    if (e < E) {
#pragma unroll
        for (int r = 0; r < kPlanCtas; ++r) {
            const int v = *cl.map_shared_rank(&s_tot[e], r);
            before += r < rank ? v : 0;
            all += v;
        }
    }
    cg::cluster_group::arrival_token left = cl.barrier_arrive();  // s_tot has been read; waited for at the end
    int total;
    const int off = block_exclusive(all, s_ws, &total);
    if (e < E) {
        int at = off + before;
#pragma unroll
        for (int w = 0; w < 32; ++w) {
            s_cnt[w * E + e] = at;
            at += c[w];
        }
        if (rank == 0) {
            counts[e] = all;
            offsets[e] = off;
        }
    }
    if (rank == 0 && e == 0) offsets[E] = total;
    for (int64_t i = total + rank * 1024 + threadIdx.x; i < n; i += kPlanCtas * 1024) perm_tok[i] = -1;
    __syncthreads();
    for (int64_t i = i0; i - lane < i1; i += 32 * kPlanBatch) {
        if (run > 32 * kPlanBatch) load_ids(idx, i, i1, E, id);
        unsigned same[kPlanBatch];
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) same[j] = same_id(id[j], bits);
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) {
            const int64_t at = i + 32 * j;
            const int earlier = __popc(same[j] & ((1u << lane) - 1u));
            const int p = id[j] >= 0 ? cnt[id[j]] + earlier : -1;
            __syncwarp();
            if (id[j] >= 0 && earlier == 0) cnt[id[j]] += __popc(same[j]);
            __syncwarp();
            if (at < i1) pos_of[at] = p;
        }
    }
    cl.barrier_wait(std::move(left));  // no CTA leaves while another reads its s_tot
}

// perm_tok of the kept lanes, one thread a lane (a plan without rows)
__global__ void __launch_bounds__(256) perm_tok_kernel(const int32_t *__restrict__ pos_of, int n, int k,
                                                       int32_t *__restrict__ perm_tok) {
    pdl_wait_then_release();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n && pos_of[i] >= 0) perm_tok[pos_of[i]] = i / k;
}

// The token's row to each of its positions, and perm_tok there, one CTA a token.  T = 8192, k = 8, H = 6144
// bf16: 158 us with the plan, 5.74 TB/s of rows; 171 without the early load of x.
template <typename V>
__global__ void __launch_bounds__(256) permute_rows_kernel(const int32_t *__restrict__ pos_of, int k,
                                                           const void *__restrict__ x, void *__restrict__ xs,
                                                           int64_t nv, int32_t *__restrict__ perm_tok) {
    __shared__ int s_pos[32];
    const int64_t t = blockIdx.x;
    RowCopy<V> row;
    row.load(x, t, nv);  // x is not the plan kernel's output, and was complete when that kernel began
    pdl_wait_then_release();
    if (threadIdx.x < k) {
        const int p = pos_of[t * k + threadIdx.x];
        s_pos[threadIdx.x] = p;
        if (p >= 0) perm_tok[p] = (int)t;
    }
    __syncthreads();
    row.store(x, xs, t, nv, s_pos, k);
}

template <typename V>
int permute_launch(const int32_t *idx, int64_t T, int k, int E, const void *x, void *xs, int64_t nv, int32_t *counts,
                   int32_t *offsets, int32_t *perm_tok, int32_t *pos_of, cudaStream_t st) {
    const int64_t n = T * k;
    if (n <= kSmallLanes) {
        VF_CUDA(launch_pdl(permute_small_kernel<V>, dim3((unsigned)T + 1), dim3(256), 0, st, idx, (int)T, k, E, x, xs,
                           nv, counts, offsets, perm_tok, pos_of));
        VF_LAUNCH_CHECK("permute_small_kernel");
        return VFMOE_OK;
    }
    const int smem = 32 * E * (int)sizeof(int);
    const int rc = set_smem_attr_once(reinterpret_cast<const void *>(plan_kernel), 32 * 1024 * (int)sizeof(int));
    if (rc) return rc;
    plan_kernel<<<kPlanCtas, 1024, smem, st>>>(idx, n, k, E, counts, offsets, perm_tok, pos_of);
    VF_LAUNCH_CHECK("plan_kernel");
    if (!x) {
        VF_CUDA(launch_pdl(perm_tok_kernel, dim3((unsigned)cdiv(n, 256)), dim3(256), 0, st, pos_of, (int)n, k, perm_tok));
        VF_LAUNCH_CHECK("perm_tok_kernel");
        return VFMOE_OK;
    }
    VF_CUDA(launch_pdl(permute_rows_kernel<V>, dim3((unsigned)T), dim3(row_threads(nv)), 0, st, pos_of, k, x, xs, nv,
                       perm_tok));
    VF_LAUNCH_CHECK("permute_rows_kernel");
    return VFMOE_OK;
}

// ----------------------------------------------------------------------------- way back
// A token's lanes that have a row, in lane order: first element of the row in y, weight, lane.  Written by
// the CTA's first warp (k <= 32); the loops below then run over rows without a branch among their loads.
struct KeptRows {
    int64_t at[32];
    float w[32];
    int lane[32];
    int n;
};

__device__ __forceinline__ void find_rows(KeptRows &s, const int32_t *pos_of, const float *w, int64_t t, int k,
                                          int64_t H) {
    if (threadIdx.x < 32) {
        const int l = threadIdx.x;
        const int32_t p = l < k ? pos_of[t * k + l] : -1;
        const float wl = l < k && w ? w[t * k + l] : 1.0f;
        const unsigned m = __ballot_sync(0xffffffffu, p >= 0);
        if (p >= 0) {
            const int i = __popc(m & ((1u << l) - 1u));
            s.at[i] = (int64_t)p * H;
            s.w[i] = wl;
            s.lane[i] = l;
        }
        if (l == 0) s.n = __popc(m);
    }
    __syncthreads();
}

// acc += w * y over U rows, their loads in flight together
template <int DT, int VE, int U>
__device__ __forceinline__ void add_rows(const KeptRows &s, int i, const void *__restrict__ y, int64_t c,
                                         float (&acc)[VE]) {
    Vec<DT, VE> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = ldv<DT, VE>(y, s.at[i + u] + c);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VE; ++j) acc[j] = fmaf(s.w[i + u], to_f32<DT>(v[u].e[j]), acc[j]);
}

// out[t] = sum_l w[t,l] y[pos_of[t,l]] (+ y_shared[t]); one thread owns VE columns and adds the lanes in order.
template <int DT, int VE>
__global__ void __launch_bounds__(256) return_rows_kernel(const void *__restrict__ y, const int32_t *__restrict__ pos_of,
                                                          const float *__restrict__ w, int64_t H, int k,
                                                          const void *__restrict__ y_shared, void *__restrict__ out,
                                                          int out_dtype) {
    __shared__ KeptRows s;
    pdl_wait_then_release();
    const int64_t t = blockIdx.x;
    find_rows(s, pos_of, w, t, k, H);
    for (int64_t c = (blockIdx.y * (int64_t)blockDim.x + threadIdx.x) * VE; c < H;
         c += (int64_t)gridDim.y * blockDim.x * VE) {
        float acc[VE] = {};
        int i = 0;
        for (; i + 8 <= s.n; i += 8) add_rows<DT, VE, 8>(s, i, y, c, acc);
        if (i + 4 <= s.n) {
            add_rows<DT, VE, 4>(s, i, y, c, acc);
            i += 4;
        }
        for (; i < s.n; ++i) add_rows<DT, VE, 1>(s, i, y, c, acc);
        if (y_shared) {
            const Vec<DT, VE> v = ldv<DT, VE>(y_shared, t * H + c);
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += to_f32<DT>(v.e[j]);
        }
        stv_dt<VE>(out, t * H + c, acc, out_dtype);
    }
}

// U rows of the gradient: dy = w dout, dot products of dout and y into s_dot[warp][row]
template <int DT, int VE, int U>
__device__ __forceinline__ void backward_rows(const KeptRows &s, int i, const void *dout, int dout_dtype, int64_t t,
                                              const void *y, int64_t H, void *dy, bool want_dw, float *s_dot) {
    float dot[U] = {};
    for (int64_t c = (int64_t)threadIdx.x * VE; c < H; c += (int64_t)blockDim.x * VE) {
        Vec<DT, VE> v[U];
        if (want_dw) {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = ldv<DT, VE>(y, s.at[i + u] + c);
        }
        float d[VE];
        ldv_dt<VE>(dout, t * H + c, d, dout_dtype);
        if (want_dw) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < VE; ++j) dot[u] = fmaf(d[j], to_f32<DT>(v[u].e[j]), dot[u]);
        }
        if (dy) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float o[VE];
#pragma unroll
                for (int j = 0; j < VE; ++j) o[j] = s.w[i + u] * d[j];
                stv<DT, VE>(dy, s.at[i + u] + c, o);
            }
        }
    }
    if (!want_dw) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float sum = warp_sum_f32(dot[u]);
        if ((threadIdx.x & 31) == 0) s_dot[(threadIdx.x >> 5) * 32 + i + u] = sum;
    }
}

// dy[pos] = w dout[t] and dw = <dout[t], y[pos]>, one CTA a token, kept rows in groups: a thread loads the
// group's columns of y together before it writes them (so dy may be y).
template <int DT, int VE>
__global__ void __launch_bounds__(256) combine_backward_kernel(const void *dout, int dout_dtype, const void *y,
                                                               const int32_t *__restrict__ pos_of,
                                                               const float *__restrict__ w, int64_t H, int k, void *dy,
                                                               float *__restrict__ dw) {
    __shared__ KeptRows s;
    __shared__ float s_dot[8 * 32];
    pdl_wait_then_release();
    const int64_t t = blockIdx.x;
    find_rows(s, pos_of, w, t, k, H);
    // rows in flight a thread: T = 8192, k = 8, H = 6144 bf16 took 269 us with 2 rows, 298 with 4, 302 with 8
    // (registers); T = 4096, H = 2048 fp32 92.7 / 90.2 / 89.2; T = 8192, H = 1001 bf16 by elements 128 / 101 / 88
    constexpr int U = VE == 1 ? 8 : VE == 4 ? 4 : 2;
    int i = 0;
    for (; i + U <= s.n; i += U) backward_rows<DT, VE, U>(s, i, dout, dout_dtype, t, y, H, dy, dw, s_dot);
    if (U == 8 && i + 4 <= s.n) {
        backward_rows<DT, VE, 4>(s, i, dout, dout_dtype, t, y, H, dy, dw, s_dot);
        i += 4;
    }
    for (; i < s.n; ++i) backward_rows<DT, VE, 1>(s, i, dout, dout_dtype, t, y, H, dy, dw, s_dot);
    if (!dw) return;
    if (threadIdx.x < k) dw[t * k + threadIdx.x] = 0.f;
    __syncthreads();
    if (threadIdx.x < s.n) {
        float sum = 0.f;
        for (int u = 0; u < (int)(blockDim.x >> 5); ++u) sum += s_dot[u * 32 + threadIdx.x];
        dw[t * k + s.lane[threadIdx.x]] = sum;
    }
}

template <int DT, int VE>
int return_launch(const void *y, const int32_t *pos_of, const float *w, int64_t T, int64_t H, int k,
                  const void *y_shared, void *out, int out_dtype, cudaStream_t st) {
    const unsigned th = row_threads(H / VE);
    const int64_t cols = cdiv(H / VE, th);
    const dim3 grid((unsigned)T, (unsigned)(cols < 65535 ? cols : 65535));
    VF_CUDA(launch_pdl(return_rows_kernel<DT, VE>, grid, dim3(th), 0, st, y, pos_of, w, H, k, y_shared, out, out_dtype));
    VF_LAUNCH_CHECK("return_rows_kernel");
    return VFMOE_OK;
}

template <int DT, int VE>
int combine_backward_launch(const void *dout, int dout_dtype, const void *y, const int32_t *pos_of, const float *w,
                            int64_t T, int64_t H, int k, void *dy, float *dw, cudaStream_t st) {
    VF_CUDA(launch_pdl(combine_backward_kernel<DT, VE>, dim3((unsigned)T), dim3(row_threads(H / VE)), 0, st, dout,
                       dout_dtype, y, pos_of, w, H, k, dy, dw));
    VF_LAUNCH_CHECK("combine_backward_kernel");
    return VFMOE_OK;
}

inline bool aligned(const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

// Rows move as 16-byte words where their length and both addresses allow, else element by element.
int launch_permute(const int32_t *idx, int64_t T, int k, int E, const void *x, int dtype, int64_t H, void *xs,
                   int32_t *counts, int32_t *offsets, int32_t *perm_tok, int32_t *pos_of, cudaStream_t st) {
    const int64_t bytes = H * elem_size(dtype);
    if (bytes % 16 == 0 && aligned(x, 16) && aligned(xs, 16))
        return permute_launch<uint4>(idx, T, k, E, x, xs, bytes / 16, counts, offsets, perm_tok, pos_of, st);
    if (elem_size(dtype) == 4)
        return permute_launch<uint32_t>(idx, T, k, E, x, xs, H, counts, offsets, perm_tok, pos_of, st);
    return permute_launch<uint16_t>(idx, T, k, E, x, xs, H, counts, offsets, perm_tok, pos_of, st);
}

// 16-byte words of y (8 columns of a 16-bit type, 4 of fp32) where rows and addresses allow, else 8-byte words of a 16-bit
// type, else columns.  All forms add in the same order, so the bits are the same.  Few rows of a 16-bit type go in 8-byte words
// too (twice the threads, half of each one's loads to wait for).  Many rows in words of four columns take the layer's
// combine_kernel (32 registers a thread against 43, CTAs of 1,024 columns), where they fill its CTAs and k leaves at most three
// lanes to its loop of eight, which takes a remainder one lane at a time.  B200, bf16 out with shared rows, us (inputs larger
// than L2 at T = 4096):
//   fp16, H = 6144, k = 8: T = 1 8-byte words 1.86, 16-byte 2.38;  T = 4096 94.1, 83.9
//   fp16, H = 1020, T = 4096: k = 8 combine_kernel 18.1, 8-byte words 18.8, columns 40.8;  k = 6 20.5, 17.2, 52.9
//   fp32, H = 6144, T = 4096: k = 2 combine_kernel 64.3, 16-byte words 77.2;  k = 8 141, 151;  k = 6 131, 130
//   fp32, T = 32, H = 6144, k = 6: 2.82, 2.18;  T = 4096, H = 512, k = 6: 16.2, 12.6
int launch_return_rows(const void *y, int y_dtype, const int32_t *pos_of, const float *w, int64_t T, int64_t H, int k,
                       const void *y_shared, void *out, int out_dtype, cudaStream_t st) {
    const int es = elem_size(y_dtype), os = elem_size(out_dtype);
    const bool many = T * H >= (int64_t)1 << 18;
    // words of n columns: the rows' length and all addresses allow them
    auto words = [&](int n) {
        return H % n == 0 && aligned(y, n * es) && aligned(y_shared, n * es) && aligned(out, n * os < 16 ? n * os : 16);
    };
    const bool full = many && H > 512 && H <= 65535 * 1024 && k % 8 < 4;
#define VF_RETURN(DT, VE) return return_launch<DT, VE>(y, pos_of, w, T, H, k, y_shared, out, out_dtype, st)
    if (y_dtype != VFMOE_DT_F32 && words(8) && many) {
        if (y_dtype == VFMOE_DT_F16) VF_RETURN(VFMOE_DT_F16, 8);
        VF_RETURN(VFMOE_DT_BF16, 8);
    }
    if (words(4)) {
        if (full && y_dtype != VFMOE_DT_BF16)
            return launch_combine(y, y_dtype, pos_of, w, (int)T, (int)H, k, y_shared, out, out_dtype, st);
        if (y_dtype == VFMOE_DT_F32) VF_RETURN(VFMOE_DT_F32, 4);
        if (y_dtype == VFMOE_DT_F16) VF_RETURN(VFMOE_DT_F16, 4);
        VF_RETURN(VFMOE_DT_BF16, 4);
    }
    if (y_dtype == VFMOE_DT_F32) VF_RETURN(VFMOE_DT_F32, 1);
    if (y_dtype == VFMOE_DT_F16) VF_RETURN(VFMOE_DT_F16, 1);
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
