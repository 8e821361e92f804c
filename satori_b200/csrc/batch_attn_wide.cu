// batch_attn_wide.cu -- attention of a batch over a paged cache with heads of more than 128 columns, on the FP32
// units.
//
// For a query row r and its visible keys t: out_r = sum_t p_rt v_t / sum_t p_rt, p_rt = 2^(s_rt - m_r),
// s_rt = (q_r . k_t) log2(e) / sqrt(d), m_r the running maximum.  One pass over the keys; the running
// maximum, the sum and the accumulator stay in FP32 registers, and each item of the plan leaves either the
// outputs or one partial record (m, sum, accumulator) per row.
//
// Two paths, by the rows of the item's tile:
//  * at most 8 rows (the query heads of one KV head of one request): each warp walks 8 keys at a time on
//    its own, K and V straight from global memory into registers; HBM bounds it.
//  * up to 64 rows (a shared prefix, a prompt): 64 x 64 tiles through shared memory, 4 x 4 scores and
//    4 x 16 outputs per thread; the FP32 units bound it.
//
// Measured with 8 heads of 256 over 2: 16 requests of 2048 to 4096 tokens 78 us in bf16 and 109 in FP32 (16 and 32 at
// the rate of HBM; loads are not asynchronous here), 64 behind 8192 shared tokens 195 and 231 us, 4 prompts of 250 to 500
// behind 2048 934 and 1018 us (396 of FP32 products at 74 TFLOP/s).
#include "batch.cuh"
#include "common.cuh"

#include <algorithm>

namespace satori {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTileM = 64, kBlock = 64, kFewRows = 8;
constexpr int HD = 256;                                // columns; those behind a smaller head's own are zeros

__device__ __forceinline__ float log2_exp(float x) { return exp2f(x); }

// 16 bytes of T as floats.
template <int TYPE>
__device__ __forceinline__ void unpack16(uint4 v, float *f)
{
    if (TYPE == SATORI_F32) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    } else {
        typedef typename Elem<TYPE>::type T;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T *p = reinterpret_cast<const T *>(&w[i]);
            f[2 * i] = Elem<TYPE>::to_float(p[0]);
            f[2 * i + 1] = Elem<TYPE>::to_float(p[1]);
        }
    }
}

template <int TYPE>
struct Smem {
    float q[kTileM][HD + 4];
    union {
        float k[kBlock][HD + 4];
        float p[kTileM][kBlock + 4];
        float few_p[kWarps][kFewRows][kFewRows];       // [warp][key][row]
        float few_o[kWarps][kFewRows][HD];
    };
    float v[kBlock][HD];
    float few_m[kWarps][kFewRows], few_l[kWarps][kFewRows];
    int limit[kTileM];                                 // visible keys of the segment, per row
    int row[kTileM];                                   // global row and query head of a tile row
    int head[kTileM];
};

// The item's rows: query values scaled by log2(e) / sqrt(d) are not rounded again (FP32), limits, indices.
template <int TYPE>
__device__ void load_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item,
                          Smem<TYPE> &sm, int rows)
{
    typedef typename Elem<TYPE>::type T;
    const PlanRow *seg_rows = plan_array<PlanRow>(plan, plan->seg_rows) + item.row_off;
    for (int r = threadIdx.x; r < rows; r += kThreads) {
        const int m = item.m0 + r;
        const bool live = r < item.m;
        const PlanRow row = live ? seg_rows[m / a.group] : PlanRow{0, 0};
        sm.row[r] = row.row;
        sm.head[r] = item.kv_head * a.group + m % a.group;
        sm.limit[r] = !live ? 0 : item.start >= 0 ? row.position + 1 - item.start : item.keys;
    }
    __syncthreads();
    const int chunks = a.head_dim / 8;
    for (int i = threadIdx.x; i < rows * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8), c = i % (HD / 8);
        float f[8] = {};
        if (r < item.m && c < chunks) {
            const T *src = reinterpret_cast<const T *>(a.q) + (long long)sm.row[r] * a.ldq +
                           (long long)sm.head[r] * a.head_dim + c * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = Elem<TYPE>::to_float(src[j]) * a.scale_log2;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sm.q[r][c * 8 + j] = f[j];
    }
    __syncthreads();
}

// Token t of the segment: its K row of the KV head; the V row lies `kv_stride` elements further.
template <typename T>
struct KeyRows {
    const T *pool;
    const int *pages;
    int shift, mask;
    long long page_elems, head_off, kv_stride;
    int head_dim;
    __device__ __forceinline__ const T *key(int t) const
    {
        return pool + (long long)pages[t >> shift] * page_elems + head_off + (long long)(t & mask) * head_dim;
    }
};

template <int TYPE>
__device__ __forceinline__ void store_out(const BatchAttn &a, int row, int head, int d, float v)
{
    const long long at = (long long)row * a.ldo + (long long)head * a.head_dim + d;
    if (a.out_f32)
        reinterpret_cast<float *>(a.out)[at] = v;
    else
        reinterpret_cast<typename Elem<TYPE>::type *>(a.out)[at] = Elem<TYPE>::from_float(v);
}

// ---- few rows: one warp, 8 keys at a time
template <int TYPE>
__device__ void few_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item,
                         const KeyRows<typename Elem<TYPE>::type> &rows, Smem<TYPE> &sm)
{
    typedef typename Elem<TYPE>::type T;
    constexpr int EV = 16 / sizeof(T);                 // elements of a 16-byte chunk
    constexpr int CH = HD / EV / 4;                    // chunks of a K row per lane (4 lanes share a key)
    constexpr int VW = HD / 32;                        // V elements per lane
    load_rows<TYPE>(a, plan, item, sm, kFewRows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = lane & 3;
    const int key0 = item.block0 * kBlock, key1 = min(key0 + item.blocks * kBlock, item.keys);
    const int chunks = a.head_dim / EV;
    int limit[kFewRows], least = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        limit[r] = sm.limit[r];
        if (r < item.m) least = min(least, limit[r]);
    }
    float m[kFewRows], l[kFewRows], acc[kFewRows][VW];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0;
#pragma unroll
        for (int j = 0; j < VW; ++j) acc[r][j] = 0;
    }
    for (int t0 = key0 + warp * 8; t0 < key1; t0 += kWarps * 8) {
        const int t = t0 + (lane >> 2);
        const bool have = t < key1;
        uint4 kc[CH];
        if (have) {
            const uint4 *src = reinterpret_cast<const uint4 *>(rows.key(t));
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (i * 4 + quarter < chunks) kc[i] = __ldg(src + i * 4 + quarter);
        }
        // V of the 8 keys: lane holds VW elements of each.
        float v[8][VW];
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            const bool use = t0 + kk < key1 && lane * VW < a.head_dim;
            const T *src = use ? rows.key(t0 + kk) + rows.kv_stride + lane * VW : nullptr;
#pragma unroll
            for (int j = 0; j < VW; ++j) v[kk][j] = 0;
            if (use) {
                if (VW * sizeof(T) >= 16) {
#pragma unroll
                    for (int j = 0; j < VW; j += EV)
                        unpack16<TYPE>(__ldg(reinterpret_cast<const uint4 *>(src + j)), &v[kk][j % VW]);
                } else {
#pragma unroll
                    for (int j = 0; j < VW; ++j) v[kk][j] = Elem<TYPE>::to_float(src[j]);
                }
            }
        }
        float s[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) s[r] = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (have && i * 4 + quarter < chunks) {
                float f[EV];
                unpack16<TYPE>(kc[i], f);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) {
                    const float *q = &sm.q[r][(i * 4 + quarter) * EV];
#pragma unroll
                    for (int j = 0; j < EV; j += 4) {
                        const float4 qv = *reinterpret_cast<const float4 *>(q + j);
                        s[r] = fmaf(qv.x, f[j], s[r]);
                        s[r] = fmaf(qv.y, f[j + 1], s[r]);
                        s[r] = fmaf(qv.z, f[j + 2], s[r]);
                        s[r] = fmaf(qv.w, f[j + 3], s[r]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            s[r] += __shfl_xor_sync(0xFFFFFFFFu, s[r], 1);
            s[r] += __shfl_xor_sync(0xFFFFFFFFu, s[r], 2);
            if (t >= limit[r] || !have) s[r] = -INFINITY;
            float top = s[r];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            top = fmaxf(top, m[r]);
            const float base = top == -INFINITY ? 0.0f : top;
            const float keep = log2_exp(m[r] - base);
            const float p = log2_exp(s[r] - base);
            m[r] = top;
            l[r] = fmaf(l[r], keep, p);                // this lane's key only; lanes are added at the end
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[r][j] *= keep;
            if (quarter == 0) sm.few_p[warp][lane >> 2][r] = p;
        }
        __syncwarp();
        const bool masked = t0 + 8 > least;            // some row of the item does not see some of these keys
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            const float4 pa = *reinterpret_cast<const float4 *>(&sm.few_p[warp][kk][0]);
            const float4 pb = *reinterpret_cast<const float4 *>(&sm.few_p[warp][kk][4]);
            const float p[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                if (masked && t0 + kk >= limit[r]) continue;       // whatever V holds there
#pragma unroll
                for (int j = 0; j < VW; ++j) acc[r][j] = fmaf(p[r], v[kk][j], acc[r][j]);
            }
        }
        __syncwarp();
    }
    // Merge the warps.
#pragma unroll
    for (int r = 0; r < kFewRows; ++r)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], o);
    __syncthreads();                                   // few_p and few_o share memory
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        if (lane == 0) {
            sm.few_m[warp][r] = m[r];
            sm.few_l[warp][r] = l[r];
        }
#pragma unroll
        for (int j = 0; j < VW; ++j) sm.few_o[warp][r][lane * VW + j] = acc[r][j];
    }
    __syncthreads();
    const int r = warp;                                // warp r merges row r
    if (r < item.m) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.few_m[w][r]);
        const float base = top == -INFINITY ? 0.0f : top;
        float weight[kWarps], sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            weight[w] = log2_exp(sm.few_m[w][r] - base);
            sum = fmaf(sm.few_l[w][r], weight[w], sum);
        }
        for (int d = lane; d < a.head_dim; d += 32) {
            float o = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) o = fmaf(sm.few_o[w][r][d], weight[w], o);
            if (item.direct)
                store_out<TYPE>(a, sm.row[r], sm.head[r], d, o / sum);
            else
                plan->part_o[((long long)item.slot * kTileM + r) * a.head_dim + d] = o;
        }
        if (!item.direct && lane == 0) plan->part_ml[(long long)item.slot * kTileM + r] = make_float2(top, sum);
    }
    __syncthreads();
}

// ---- many rows: 64 x 64 tiles
template <int TYPE>
__device__ void many_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item,
                          const KeyRows<typename Elem<TYPE>::type> &rows, Smem<TYPE> &sm)
{
    typedef typename Elem<TYPE>::type T;
    constexpr int EV = 16 / sizeof(T);
    constexpr int OC = HD / 64;                        // float4 groups of output columns per thread
    load_rows<TYPE>(a, plan, item, sm, kTileM);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int chunks = a.head_dim / EV;
    float m[4], l[4], acc[4][OC * 4];
    int limit[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        limit[i] = sm.limit[ty * 4 + i];
        m[i] = -INFINITY;
        l[i] = 0;
#pragma unroll
        for (int j = 0; j < OC * 4; ++j) acc[i][j] = 0;
    }
    const int least = sm.limit[0];                     // keys that every row of the tile sees
    for (int block = item.block0; block < item.block0 + item.blocks; ++block) {
        const int t0 = block * kBlock, have = min(kBlock, item.keys - t0);
        for (int i = threadIdx.x; i < kBlock * (HD / EV); i += kThreads) {
            const int t = i / (HD / EV), c = i % (HD / EV);
            float fk[EV], fv[EV];
#pragma unroll
            for (int j = 0; j < EV; ++j) fk[j] = fv[j] = 0;
            if (t < have && c < chunks) {
                const T *src = rows.key(t0 + t) + c * EV;
                unpack16<TYPE>(__ldg(reinterpret_cast<const uint4 *>(src)), fk);
                unpack16<TYPE>(__ldg(reinterpret_cast<const uint4 *>(src + rows.kv_stride)), fv);
            }
#pragma unroll
            for (int j = 0; j < EV; j += 4) {
                *reinterpret_cast<float4 *>(&sm.k[t][c * EV + j]) = make_float4(fk[j], fk[j + 1], fk[j + 2], fk[j + 3]);
                *reinterpret_cast<float4 *>(&sm.v[t][c * EV + j]) = make_float4(fv[j], fv[j + 1], fv[j + 2], fv[j + 3]);
            }
        }
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0;
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            float4 q[4], k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4 *>(&sm.q[ty * 4 + i][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4 *>(&sm.k[tx + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
                    s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
                    s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
                    s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
                }
        }
        __syncthreads();                               // k is done: p takes its place
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (t0 + tx + 16 * j >= limit[i]) s[i][j] = -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const float base = top == -INFINITY ? 0.0f : top;
            const float keep = log2_exp(m[i] - base);
            m[i] = top;
            float sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = log2_exp(s[i][j] - base);
                sum += p;
                sm.p[ty * 4 + i][tx + 16 * j] = p;
            }
            l[i] = fmaf(l[i], keep, sum);              // this thread's keys only
#pragma unroll
            for (int j = 0; j < OC * 4; ++j) acc[i][j] *= keep;
        }
        __syncthreads();
        const bool masked = t0 + kBlock > least;       // some row does not see some key of the block
#pragma unroll 2
        for (int t = 0; t < kBlock; t += 4) {
            float4 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4 *>(&sm.p[ty * 4 + i][t]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int c = 0; c < OC; ++c) {
                    const float4 v = *reinterpret_cast<const float4 *>(&sm.v[t + u][c * 64 + tx * 4]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                        if (masked && t0 + t + u >= limit[i]) continue;        // whatever V holds there
                        acc[i][c * 4] = fmaf(w, v.x, acc[i][c * 4]);
                        acc[i][c * 4 + 1] = fmaf(w, v.y, acc[i][c * 4 + 1]);
                        acc[i][c * 4 + 2] = fmaf(w, v.z, acc[i][c * 4 + 2]);
                        acc[i][c * 4 + 3] = fmaf(w, v.w, acc[i][c * 4 + 3]);
                    }
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], o);
        const int r = ty * 4 + i;
        if (r < item.m) {
            const float inverse = 1.0f / l[i];
#pragma unroll
            for (int c = 0; c < OC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = c * 64 + tx * 4 + j;
                    if (d < a.head_dim) {
                        if (item.direct)
                            store_out<TYPE>(a, sm.row[r], sm.head[r], d, acc[i][c * 4 + j] * inverse);
                        else
                            plan->part_o[((long long)item.slot * kTileM + r) * a.head_dim + d] = acc[i][c * 4 + j];
                    }
                }
            if (!item.direct && tx == 0) plan->part_ml[(long long)item.slot * kTileM + r] = make_float2(m[i], l[i]);
        }
    }
    __syncthreads();
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads, 1) wide_attention_kernel(const BatchAttn a)
{
    typedef typename Elem<TYPE>::type T;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem<TYPE> &sm = *reinterpret_cast<Smem<TYPE> *>(smem_raw);
    pdl_launch_dependents();
    pdl_wait();
    const DevPlan *plan = a.plan;
    const int *cta_off = plan_array<int>(plan, plan->cta_off);
    KeyRows<T> rows;
    rows.pool = reinterpret_cast<const T *>(a.pool);
    rows.shift = __ffs(a.page_tokens) - 1;
    rows.mask = a.page_tokens - 1;
    rows.head_dim = a.head_dim;
    rows.kv_stride = (long long)a.kv_heads * a.page_tokens * a.head_dim;
    rows.page_elems = 2 * rows.kv_stride;
    for (int i = cta_off[blockIdx.x]; i < cta_off[blockIdx.x + 1]; ++i) {
        const PlanItem item = plan_array<PlanItem>(plan, plan->items)[i];
        rows.pages = plan_array<int>(plan, plan->pages) + item.page_off;
        rows.head_off = (long long)item.kv_head * a.page_tokens * a.head_dim;
        if (item.m <= kFewRows)
            few_rows<TYPE>(a, plan, item, rows, sm);
        else
            many_rows<TYPE>(a, plan, item, rows, sm);
    }
}

template <int TYPE>
cudaError_t launch(const BatchAttn &a, cudaStream_t stream)
{
    cudaError_t e = opt_in_smem(reinterpret_cast<const void *>(&wide_attention_kernel<TYPE>), sizeof(Smem<TYPE>));
    if (e != cudaSuccess) return e;
    return launch_overlapped(wide_attention_kernel<TYPE>, dim3(a.ctas), kThreads, sizeof(Smem<TYPE>), stream, a);
}

}  // namespace

void wide_plan_shape(int sm_count, PlanShape &shape)
{
    shape.tile_m = kTileM;
    shape.block = kBlock;
    shape.ctas = sm_count;
    shape.solo_m = kFewRows;
    // A block of 64 keys costs the small path about half of what the 64-row path needs.
    shape.solo_cost = 2;
    shape.pair_cost = 4;
    shape.item_cost = 2;
    shape.slots_per_item = 1;
}

int wide_record_rows() { return kTileM; }

cudaError_t launch_wide_attention(const BatchAttn &a, cudaStream_t stream)
{
    switch (a.type) {
    case SATORI_F32: return launch<SATORI_F32>(a, stream);
    case SATORI_F16: return launch<SATORI_F16>(a, stream);
    default: return launch<SATORI_BF16>(a, stream);
    }
}

}  // namespace satori
