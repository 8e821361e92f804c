// batch.cu -- a decode batch over a paged cache: its C ABI, the append of the new tokens, and the merge of
// partial attention records.
//
// A step plans once on the host what every layer repeats: where each new token goes, and which keys are read
// for which rows together.  The plan is uploaded behind one device pointer that never moves while it fits, so
// the launches of a step's layers can be captured and replayed for the next steps.
#include "batch.cuh"
#include "common.cuh"
#include "paged_internal.h"
#include "staging.h"

#include <math.h>
#include <string.h>

#include <algorithm>

using namespace satori;

struct satori_batch {
    satori_pages *pages = nullptr;
    int q_heads = 0, rotary = 0;
    double rope_base = 0;
    PlanShape shape = {};
    Plan plan;
    struct Member {
        int id;
        unsigned version;
    };
    std::vector<Member> members;
    bool planned = false;
    int reallocations = 0;                     // times that the plan moved: earlier captures repeat an old step
    // Device buffers; one that grows leaves the old one allocated, so that a graph captured before finds
    // valid memory (of an old step) and no freed one.
    int *d_plan = nullptr;
    size_t plan_ints = 0;
    uint8_t *d_partials = nullptr;             // [records][rows][dim] floats, then [records][rows] (max, sum)
    size_t partials = 0;
    double *d_rope = nullptr;                  // [row][rotary / 2] (cos, sin)
    size_t rope_rows = 0;
    std::vector<void *> outgrown;
    Staging staging;
};

namespace {

template <typename V>
int place(std::vector<V> const &v, size_t &at)
{
    at = (at + 3) / 4 * 4;                     // 16-byte aligned arrays
    const int here = (int)at;
    at += v.size() * sizeof(V) / 4;
    return here;
}

template <typename V>
void put(int *base, int at, std::vector<V> const &v)
{
    if (!v.empty()) memcpy(base + at, v.data(), v.size() * sizeof(V));
}

// ------------------------------------------------------------------------------------------- kernels

// The step's RoPE factors: (cos, sin) of TransformerOps.RopeHalf's FP64 angle (TransformerOps.cs:99-118) for
// every row and pair, the same for every head and layer.
__global__ void rope_rows_kernel(const DevPlan *plan, double base, int rotary, double *table)
{
    const int half = rotary / 2, n = plan->head.rows * half;
    const int *position = plan_array<int>(plan, plan->row_position);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const int row = i / half, k = i % half;
        const double angle = __ddiv_rn((double)position[row], pow(base, __ddiv_rn(2.0 * k, (double)rotary)));
        double sn, cs;
        sincos(angle, &sn, &cs);
        table[2 * (size_t)i] = cs;
        table[2 * (size_t)i + 1] = sn;
    }
}

struct AppendArgs {
    const DevPlan *plan;
    const void *q, *k, *v;                     // rows ldq / ldk / ldv elements apart; q may be null
    long long ldq, ldk, ldv;
    void *q_out;                               // [rows][q_heads * head_dim]
    uint8_t *pool;                             // the layer's pages
    int q_heads, kv_heads, head_dim, rotary, page_tokens;
};

// Loads and stores of 4 values; `wide`: the rows are aligned for one access.  (Ordinary loads, not the read-only
// path: q may be rotated in place.)
template <int TYPE>
__device__ __forceinline__ void load4(const typename Elem<TYPE>::type *p, bool wide, float *f)
{
    typedef typename Elem<TYPE>::type T;
    union {
        T t[4];
        float4 f4;
        uint2 u2;
    } v;
    if (wide) {
        if (TYPE == SATORI_F32)
            v.f4 = *reinterpret_cast<const float4 *>(p);
        else
            v.u2 = *reinterpret_cast<const uint2 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v.t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = Elem<TYPE>::to_float(v.t[i]);
}

template <int TYPE>
__device__ __forceinline__ void store4(typename Elem<TYPE>::type *p, bool wide, const typename Elem<TYPE>::type *t)
{
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = t[i];
    } else if (TYPE == SATORI_F32) {
        *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(t);
    } else {
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(t);
    }
}

// One thread turns 8 values of one (row, head): two runs of 4, `rotary / 2` apart where they rotate
// (RopeHalf pairs i and i + rotary / 2), together where they do not.  The products are FP64 like
// RopeHalf's, rounded once to the output's type.  Bytes bound it: every value is read and written once.
template <int IN, int TYPE>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a, int wide_in, int wide_out)
{
    typedef typename Elem<IN>::type TI;
    typedef typename Elem<TYPE>::type T;
    const DevPlan *plan = a.plan;
    const int chunks = a.head_dim / 8, heads = (a.q ? a.q_heads : 0) + 2 * a.kv_heads;
    const long long n = (long long)plan->head.rows * heads * chunks;
    const int *page = plan_array<int>(plan, plan->row_page), *slot = plan_array<int>(plan, plan->row_slot);
    const long long kv_stride = (long long)a.kv_heads * a.page_tokens * a.head_dim;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int c = (int)(i % chunks);
        const long long j = i / chunks;
        int h = (int)(j % heads);
        const int row = (int)(j / heads);
        const TI *src;
        T *dst;
        bool rotates = true, wide = wide_out;
        if (a.q && h < a.q_heads) {
            src = (const TI *)a.q + row * a.ldq + (long long)h * a.head_dim;
            dst = (T *)a.q_out + ((long long)row * a.q_heads + h) * a.head_dim;
        } else {
            if (a.q) h -= a.q_heads;
            const bool value = h >= a.kv_heads;
            if (value) h -= a.kv_heads;
            src = value ? (const TI *)a.v + row * a.ldv + (long long)h * a.head_dim
                        : (const TI *)a.k + row * a.ldk + (long long)h * a.head_dim;
            dst = (T *)a.pool + (2ll * page[row] + value) * kv_stride + (long long)h * a.page_tokens * a.head_dim +
                  (long long)slot[row] * a.head_dim;
            rotates = !value;
            wide = true;
        }
        const int half = a.rotary / 2;
        rotates = rotates && c < a.rotary / 8;
        const int at = rotates ? 4 * c : 8 * c, step = rotates ? half : 4;
        float x[4], y[4];
        load4<IN>(src + at, wide_in, x);
        load4<IN>(src + at + step, wide_in, y);
        alignas(16) T ox[4], oy[4];
        if (rotates) {
            const double2 *cs = reinterpret_cast<const double2 *>(plan->rope) + (long long)row * half + 4 * c;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double2 f = __ldg(cs + e);
                ox[e] = Elem<TYPE>::from_double(__dsub_rn(__dmul_rn(x[e], f.x), __dmul_rn(y[e], f.y)));
                oy[e] = Elem<TYPE>::from_double(__dadd_rn(__dmul_rn(x[e], f.y), __dmul_rn(y[e], f.x)));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ox[e] = Elem<TYPE>::from_float(x[e]);
                oy[e] = Elem<TYPE>::from_float(y[e]);
            }
        }
        store4<TYPE>(dst + at, wide, ox);
        store4<TYPE>(dst + at + step, wide, oy);
    }
}

// A record's weight from its (maximum, sum).  A maximum of minus infinity: no key, and nothing was stored (sum 0), or
// none but scores of NaN (sum NaN), which the row keeps.
__device__ __forceinline__ float record_weight(float2 ml, float ref)
{
    return ml.x == -INFINITY ? ml.y : exp2f(ml.x - ref);
}

struct CombineShape {
    int record_rows, tile_m, by_column, octets, parts;
};

// out = sum_i w_i acc_i / sum_i w_i l_i with w_i = 2^(m_i - m), over the records of all the row's segments in a
// fixed order, so the result does not depend on scheduling; m is the running maximum, raised from one chunk of
// records to the next.  A block takes one row, up to 8 query heads of a KV head (their values lie side by side
// in the records) and 256 / SLICES groups of 4 values: a warp per head finds its records and their weights,
// then each slice of the threads adds every SLICES-th record, and the slices are added.  Latency bounds it
// (half a dozen loads one after the other before the first value), so loads go out 8 at a time.
constexpr int kCombineThreads = 256, kCombineHeads = 8, kCombineChunk = 64, kCombineLinks = 32;
constexpr int kCombineParts = kCombineHeads * (256 / 4) / (kCombineThreads / 4);       // of an octet's values, at most

template <int TYPE, int SLICES>
__global__ void __launch_bounds__(kCombineThreads, 4) combine_kernel(const BatchAttn a, const CombineShape c)
{
    constexpr int kCombineQuads = kCombineThreads / SLICES, kBatch = 8;
    __shared__ int first[kCombineLinks][kCombineHeads], records[kCombineLinks][kCombineHeads], step[kCombineLinks][kCombineHeads];
    __shared__ unsigned base[kCombineHeads][kCombineChunk];        // record * rows + row
    __shared__ float weight[kCombineHeads][kCombineChunk], factor[kCombineHeads], total[kCombineHeads];
    __shared__ int count[kCombineHeads];
    __shared__ float4 slices[SLICES][kCombineQuads];
    // What it reads before pdl_wait is the plan's, which lay there when the attention kernel started: a copy on the
    // stream brought it, and no launch behind a copy starts before it.  And no early start for the next launch: its
    // blocks would take the SMs from this one's.
    const DevPlan *plan = a.plan;
    const int tid = threadIdx.x, mine = tid >> 5, lane = tid & 31;
    const int quads = a.head_dim / 4;
    const int *chain_off = plan_array<int>(plan, plan->chain_off);
    const PlanLink *chain = plan_array<PlanLink>(plan, plan->chain);
    const PlanSlots *slots = plan_array<PlanSlots>(plan, plan->slots);
    const float4 *values = reinterpret_cast<const float4 *>(plan->part_o);
    const float2 *part_ml = plan->part_ml;
    const int *merges = plan_array<int>(plan, plan->merges);
    const int units = plan->head.merges * c.octets * c.parts;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        int rest = u;
        const int part = rest % c.parts;
        rest /= c.parts;
        const int g0 = rest % c.octets * kCombineHeads, heads = min(kCombineHeads, a.group - g0);
        rest /= c.octets;
        const int merge = merges[rest], kv_head = merge % a.kv_heads, row = merge / a.kv_heads;
        const int c0 = chain_off[row], c1 = chain_off[row + 1];
        // This thread's output: 4 values of one head.
        const int slice = tid / kCombineQuads, i = part * kCombineQuads + tid % kCombineQuads;
        const bool works = i < heads * quads;
        const int g = works ? (c.by_column ? i % heads : i / quads) : 0, quad = c.by_column ? i / heads : i % quads;
        float4 acc = make_float4(0, 0, 0, 0);
        float ref = -INFINITY, sum = 0;                // this warp's head
        for (int link0 = c0; link0 < c1; link0 += kCombineLinks) {
            const int links = min(kCombineLinks, c1 - link0);
            if (tid < links * kCombineHeads) {
                const int k = tid / kCombineHeads, h = tid % kCombineHeads;
                const PlanLink link = chain[link0 + k];
                const int m = link.index * a.group + g0 + min(h, heads - 1), mt = m % c.tile_m;
                const PlanSlots s = slots[(link.tile0 + m / c.tile_m) * a.kv_heads + kv_head];
                // A tile's rows run on into its second record; first -1: the item wrote the output itself.
                first[k][h] = s.first < 0 ? -1 : s.first * c.record_rows + mt;
                records[k][h] = s.records / s.step;
                step[k][h] = s.step * c.record_rows;
            }
            __syncthreads();
            const bool written = first[0][mine] < 0;
            int n = 0;
            for (int k = 0; k < links; ++k) n += records[k][mine];
            if (written || mine >= heads) n = 0;
            if (lane == 0) count[mine] = written ? -1 : n;
            __syncthreads();
            int most = 0;
            for (int h = 0; h < heads; ++h) most = max(most, count[h]);
            pdl_wait();
            for (int chunk = 0; chunk < most; chunk += kCombineChunk) {
                unsigned at[kCombineChunk / 32];
                float2 ml[kCombineChunk / 32];
#pragma unroll
                for (int j = 0; j < kCombineChunk / 32; ++j) {
                    int rank = chunk + j * 32 + lane, k = 0;
                    ml[j] = make_float2(-INFINITY, 0.0f);
                    at[j] = 0;
                    if (rank < n) {
                        while (rank >= records[k][mine]) rank -= records[k++][mine];
                        at[j] = (unsigned)first[k][mine] + (unsigned)rank * (unsigned)step[k][mine];
                        ml[j] = part_ml[at[j]];
                    }
                }
                float top = ml[0].x;
#pragma unroll
                for (int j = 1; j < kCombineChunk / 32; ++j) top = fmaxf(top, ml[j].x);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                top = fmaxf(top, ref);
                const float keep = top == -INFINITY ? 1.0f : exp2f(ref - top);
                sum *= keep;
                ref = top;
#pragma unroll
                for (int j = 0; j < kCombineChunk / 32; ++j) {
                    const float w = record_weight(ml[j], ref);
                    if (w != 0) sum = fmaf(w, ml[j].y, sum);
                    weight[mine][j * 32 + lane] = w;
                    base[mine][j * 32 + lane] = at[j];
                }
                if (lane == 0) factor[mine] = keep;
                __syncthreads();
                const int end = works ? min(kCombineChunk, count[g] - chunk) : 0;
                const float scale = factor[g];
                acc.x *= scale;
                acc.y *= scale;
                acc.z *= scale;
                acc.w *= scale;
                for (int f0 = slice; f0 < end; f0 += SLICES * kBatch) {
                    float4 v[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int f = f0 + k * SLICES;
                        v[k] = make_float4(0, 0, 0, 0);
                        if (f < end && weight[g][f] != 0) {
                            const unsigned rr = base[g][f], r = rr % (unsigned)c.record_rows;
                            v[k] = values[c.by_column ? (size_t)(rr - r) * quads + (size_t)quad * c.record_rows + r
                                                      : (size_t)rr * quads + quad];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int f = f0 + k * SLICES;
                        const float w = f < end ? weight[g][f] : 0.0f;
                        acc.x = fmaf(v[k].x, w, acc.x);
                        acc.y = fmaf(v[k].y, w, acc.y);
                        acc.z = fmaf(v[k].z, w, acc.z);
                        acc.w = fmaf(v[k].w, w, acc.w);
                    }
                }
                __syncthreads();
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (lane == 0) total[mine] = sum;
        if (slice > 0) slices[slice - 1][tid % kCombineQuads] = acc;
        __syncthreads();
        if (slice == 0 && works && count[g] >= 0) {
            const float inverse = 1.0f / total[g];
            float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
            for (int k = 0; k < SLICES - 1; ++k) {
                const float4 more = slices[k][tid];
                v[0] += more.x;
                v[1] += more.y;
                v[2] += more.z;
                v[3] += more.w;
            }
            const long long to = (long long)row * a.ldo + (long long)(kv_head * a.group + g0 + g) * a.head_dim + quad * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (a.out_f32)
                    reinterpret_cast<float *>(a.out)[to + e] = v[e] * inverse;
                else
                    reinterpret_cast<typename Elem<TYPE>::type *>(a.out)[to + e] = Elem<TYPE>::from_float(v[e] * inverse);
            }
        }
        __syncthreads();
    }
    pdl_wait();                // also without a row: launches behind this one count on the attention's end
}

// The same with a warp for a row and up to 8 query heads, for launches with thousands of rows: no barriers, and the
// loads that wait for one another are those of 24 rows an SM at a time, not of 4.  Lane (s, h) finds every fourth
// record of head h; the records' weights meet in shuffles.  ITEMS: groups of 4 output values a lane.
template <int TYPE, int ITEMS>
__global__ void __launch_bounds__(kCombineThreads, ITEMS > 8 ? 2 : 3) combine_rows_kernel(const BatchAttn a, const CombineShape c)
{
    constexpr int kLanes = 32 / kCombineHeads;         // of a head
    const DevPlan *plan = a.plan;
    const int lane = threadIdx.x & 31, h = lane % kCombineHeads, quads = a.head_dim / 4;
    const int *chain_off = plan_array<int>(plan, plan->chain_off), *merges = plan_array<int>(plan, plan->merges);
    const PlanLink *chain = plan_array<PlanLink>(plan, plan->chain);
    const PlanSlots *slots = plan_array<PlanSlots>(plan, plan->slots);
    const float4 *values = reinterpret_cast<const float4 *>(plan->part_o);
    const float2 *part_ml = plan->part_ml;
    const int units = plan->head.merges * c.octets, warps = gridDim.x * (kCombineThreads / 32);
    for (int u = blockIdx.x * (kCombineThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
        const int g0 = u % c.octets * kCombineHeads, heads = min(kCombineHeads, a.group - g0);
        const int merge = merges[u / c.octets], kv_head = merge % a.kv_heads, row = merge / a.kv_heads;
        const int c0 = chain_off[row], c1 = chain_off[row + 1];
        int link = c0, rank = lane / kCombineHeads, records = 0;
        unsigned first = 0, step = 0;
        bool direct = false;                           // the item wrote the head's output itself
        auto enter = [&] {
            const PlanLink l = chain[link];
            const int m = l.index * a.group + g0 + min(h, heads - 1), mt = m % c.tile_m;
            const PlanSlots s = slots[(l.tile0 + m / c.tile_m) * a.kv_heads + kv_head];
            direct = direct || s.first < 0;
            first = (unsigned)(s.first * c.record_rows + mt);
            records = s.records / s.step;
            step = (unsigned)(s.step * c.record_rows);
        };
        enter();
        pdl_wait();
        float4 acc[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) acc[k] = make_float4(0, 0, 0, 0);
        const int n = heads * quads;
        float ref = -INFINITY, sum = 0;
        for (;;) {
            while (link < c1 && rank >= records) {
                rank -= records;
                if (++link < c1) enter();
            }
            const bool has = link < c1 && h < heads && !direct;
            if (!__any_sync(0xFFFFFFFFu, has)) break;
            const unsigned at = has ? first + (unsigned)rank * step : 0;
            const float2 ml = has ? part_ml[at] : make_float2(-INFINITY, 0.0f);
            float top = ml.x;
#pragma unroll
            for (int o = kCombineHeads; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            top = fmaxf(top, ref);
            const float keep = top == -INFINITY ? 1.0f : exp2f(ref - top);
            const float w = record_weight(ml, top);
            sum *= keep;
            if (w != 0) sum = fmaf(w, ml.y, sum);
            ref = top;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                const int i = k * 32 + lane, g = c.by_column ? i % heads : i / quads;
                const float f = __shfl_sync(0xFFFFFFFFu, keep, g);
                acc[k].x *= f;
                acc[k].y *= f;
                acc[k].z *= f;
                acc[k].w *= f;
            }
#pragma unroll 1
            for (int s = 0; s < kLanes; ++s) {
                if (!__any_sync(0xFFFFFFFFu, lane / kCombineHeads == s && w != 0)) continue;
                float4 v[ITEMS];
                float weight[ITEMS];
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    const int i = k * 32 + lane, g = c.by_column ? i % heads : i / quads, quad = c.by_column ? i / heads : i % quads;
                    weight[k] = __shfl_sync(0xFFFFFFFFu, w, s * kCombineHeads + g);
                    const unsigned rr = __shfl_sync(0xFFFFFFFFu, at, s * kCombineHeads + g), r = rr % (unsigned)c.record_rows;
                    v[k] = make_float4(0, 0, 0, 0);
                    if (i < n && weight[k] != 0)
                        v[k] = values[c.by_column ? (size_t)(rr - r) * quads + (size_t)quad * c.record_rows + r : (size_t)rr * quads + quad];
                }
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    acc[k].x = fmaf(v[k].x, weight[k], acc[k].x);
                    acc[k].y = fmaf(v[k].y, weight[k], acc[k].y);
                    acc[k].z = fmaf(v[k].z, weight[k], acc[k].z);
                    acc[k].w = fmaf(v[k].w, weight[k], acc[k].w);
                }
            }
            rank += kLanes;
        }
#pragma unroll
        for (int o = kCombineHeads; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const float inverse = 1.0f / sum;
        const unsigned written = __ballot_sync(0xFFFFFFFFu, direct);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = k * 32 + lane, g = c.by_column ? i % heads : i / quads, quad = c.by_column ? i / heads : i % quads;
            const float f = __shfl_sync(0xFFFFFFFFu, inverse, g);
            if (i >= n || (written >> g & 1u)) continue;
            const float v[4] = {acc[k].x * f, acc[k].y * f, acc[k].z * f, acc[k].w * f};
            const long long to = (long long)row * a.ldo + (long long)(kv_head * a.group + g0 + g) * a.head_dim + quad * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (a.out_f32)
                    reinterpret_cast<float *>(a.out)[to + e] = v[e];
                else
                    reinterpret_cast<typename Elem<TYPE>::type *>(a.out)[to + e] = Elem<TYPE>::from_float(v[e]);
            }
        }
    }
    pdl_wait();                // (see above)
}

// ------------------------------------------------------------------------------------------- host side

int check_batch(satori_batch *b)
{
    if (!b) return set_error(SATORI_ERR_DISPOSED, "batch is disposed");
    if (b->pages->disposed) return set_error(SATORI_ERR_DISPOSED, "the batch's paged cache is disposed");
    return SATORI_OK;
}

// The tables are still those that the step planned for.
int check_planned(satori_batch *b)
{
    int rc = check_batch(b);
    if (rc) return rc;
    if (!b->planned) return set_error(SATORI_ERR_ARGUMENT, "the batch has no step yet");
    for (const satori_batch::Member &m : b->members) {
        const PageSequence *s = b->pages->tables.find(m.id);
        if (!s || s->version != m.version)
            return set_error(SATORI_ERR_ARGUMENT, "sequence %d changed after the batch's step", m.id);
    }
    if (!b->pages->ctx) return set_error(SATORI_ERR_NOT_SUPPORTED, "the cache has no device memory");
    return SATORI_OK;
}

// A device buffer of at least `need` units of `unit` bytes; `have` is updated.
template <typename P>
cudaError_t grow(satori_batch *b, P *&buffer, size_t &have, size_t need, size_t unit, size_t least)
{
    if (need <= have) return cudaSuccess;
    const size_t count = std::max(std::max(need, 2 * have), least);
    void *fresh = nullptr;
    if (buffer) b->outgrown.reserve(b->outgrown.size() + 1);
    cudaError_t e = cudaMalloc(&fresh, count * unit);
    if (e != cudaSuccess) return e;
    if (buffer) {
        b->outgrown.push_back(buffer);
    }
    buffer = static_cast<P *>(fresh);
    have = count;
    return cudaSuccess;
}

bool on_tensor_cores(const satori_batch *b) { return tensor_attention_takes(b->pages->type, b->pages->head_dim); }
bool on_f32_tiles(const satori_batch *b) { return f32_attention_takes(b->pages->type, b->pages->head_dim); }

size_t record_rows(const satori_batch *b)
{
    return (size_t)(on_tensor_cores(b) ? tensor_record_rows() : on_f32_tiles(b) ? f32_record_rows() : wide_record_rows());
}

int upload_plan(satori_batch *b)
{
    satori_ctx *ctx = b->pages->ctx;
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    const Plan &p = b->plan;
    DevPlan head = {};
    head.head = p.head;
    size_t ints = sizeof(DevPlan) / 4;
    head.row_position = place(p.row_position, ints);
    head.row_page = place(p.row_page, ints);
    head.row_slot = place(p.row_slot, ints);
    head.chain_off = place(p.chain_off, ints);
    head.chain = place(p.chain, ints);
    head.seg_rows = place(p.seg_rows, ints);
    head.pages = place(p.pages, ints);
    head.cta_off = place(p.cta_off, ints);
    head.slots = place(p.slots, ints);
    head.items = place(p.items, ints);
    head.merges = place(p.merges, ints);
    const size_t rows = record_rows(b);
    // What the kernels count in 32 bits: records' rows, the merges' units (with a grid's stride behind the last), and
    // the pairs of the rotation's factors.
    constexpr long long kUnits = 0x7fffffff - (1 << 20);
    const long long octets = (b->shape.group + kCombineHeads - 1) / kCombineHeads;
    if (ints > 0x7fffffff || (size_t)p.partials * rows > 0x7fffffff ||
        (long long)p.merges.size() * octets * kCombineParts > kUnits || (long long)p.head.rows * (b->rotary / 2) > kUnits)
        return set_error(SATORI_ERR_NOT_SUPPORTED, "the step's plan exceeds Int32 limits");
    const size_t record = rows * ((size_t)b->pages->head_dim + 2) * 4;
    const int *old_plan = b->d_plan;
    cudaError_t e = grow(b, b->d_plan, b->plan_ints, ints, 4, 1 << 16);
    b->reallocations += old_plan && old_plan != b->d_plan;
    if (e == cudaSuccess) e = grow(b, b->d_partials, b->partials, (size_t)p.partials, record, 1);
    if (e == cudaSuccess && b->rotary)
        e = grow(b, b->d_rope, b->rope_rows, (size_t)p.head.rows, (size_t)b->rotary * 8, 64);
    if (e != cudaSuccess) return cuda_fail(e, "allocate batch buffers");
    head.part_o = reinterpret_cast<float *>(b->d_partials);
    head.part_ml = reinterpret_cast<float2 *>(head.part_o + b->partials * rows * b->pages->head_dim);
    head.rope = b->d_rope;
    void *buffer = nullptr;
    if ((e = b->staging.take(ints * 4, &buffer)) != cudaSuccess) return cuda_fail(e, "stage the step's plan");
    int *stage = static_cast<int *>(buffer);
    memcpy(stage, &head, sizeof head);
    put(stage, head.row_position, p.row_position);
    put(stage, head.row_page, p.row_page);
    put(stage, head.row_slot, p.row_slot);
    put(stage, head.chain_off, p.chain_off);
    put(stage, head.chain, p.chain);
    put(stage, head.seg_rows, p.seg_rows);
    put(stage, head.pages, p.pages);
    put(stage, head.cta_off, p.cta_off);
    put(stage, head.slots, p.slots);
    put(stage, head.items, p.items);
    put(stage, head.merges, p.merges);
    e = b->staging.send(b->d_plan, ints * 4, ctx->stream);
    if (e == cudaSuccess && b->rotary && p.head.rows) {
        const long long pairs = (long long)p.head.rows * (b->rotary / 2);
        const unsigned blocks = (unsigned)std::min<long long>((pairs + 127) / 128, 8ll * ctx->sm_count);
        rope_rows_kernel<<<blocks, 128, 0, ctx->stream>>>(reinterpret_cast<const DevPlan *>(b->d_plan), b->rope_base,
                                                         b->rotary, b->d_rope);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? SATORI_OK : cuda_fail(e, "upload the step's plan");
}

template <int IN, int TYPE>
cudaError_t launch_append(const AppendArgs &a, int rows, int wide_in, int wide_out, int sm_count, cudaStream_t stream)
{
    const long long n = (long long)rows * ((a.q ? a.q_heads : 0) + 2 * a.kv_heads) * (a.head_dim / 8);
    const unsigned blocks = (unsigned)std::max<long long>(1, std::min<long long>((n + 255) / 256, 32ll * sm_count));
    append_kernel<IN, TYPE><<<blocks, 256, 0, stream>>>(a, wide_in, wide_out);
    return cudaGetLastError();
}

}  // namespace

template <int TYPE>
static cudaError_t launch_combine_type(const BatchAttn &a, const CombineShape &c, int slices, dim3 grid, cudaStream_t stream)
{
    if (slices == 0) {       // a warp for a row
        const int items = (std::min(a.group, kCombineHeads) * a.head_dim / 4 + 31) / 32;
        auto kernel = items <= 4 ? combine_rows_kernel<TYPE, 4> : items <= 8 ? combine_rows_kernel<TYPE, 8> : combine_rows_kernel<TYPE, 16>;
        return launch_overlapped(kernel, grid, kCombineThreads, 0, stream, a, c);
    }
    auto kernel = slices == 4 ? combine_kernel<TYPE, 4> : slices == 2 ? combine_kernel<TYPE, 2> : combine_kernel<TYPE, 1>;
    return launch_overlapped(kernel, grid, kCombineThreads, 0, stream, a, c);
}

cudaError_t satori::launch_combine(const BatchAttn &a, int record_rows, int tile_m, bool by_column, int merges, int sm_count,
                                   cudaStream_t stream)
{
    // From 2048 rows of a KV head on there are enough for a warp each (the prompts of 8 requests, 10k rows: the call
    // 137 us, with a block for each 172; 512 requests over 8 KV heads 235 and 247, 64 over 32 KV heads 134 and 138);
    // with fewer, their records are better dealt to whole blocks (256 requests over 4 KV heads 83 us, with a warp
    // for each 99; 64 behind 32k tokens 81 and 132).  There as many slices as a row's values leave threads for, and
    // more while all blocks are resident (4 an SM): one sequence of 4k tokens over 4 KV heads, 66 records a row, takes
    // 13 us with one slice, 9 with four; the call of 64 requests behind 32k tokens 66.5 us with one, 62.9 with two.
    const int outputs = std::min(a.group, kCombineHeads) * a.head_dim / 4, octets = (a.group + kCombineHeads - 1) / kCombineHeads;
    const long long rows = (long long)merges * octets;
    const bool warps = rows >= 2048;
    auto fits = [&](int slices) { return rows * ((outputs * slices + kCombineThreads - 1) / kCombineThreads) <= 4 * sm_count; };
    const int slices = warps ? 0 : outputs <= 64 || fits(4) ? 4 : outputs <= 128 || fits(2) ? 2 : 1;
    const int quads = warps ? outputs : kCombineThreads / slices;
    const CombineShape c = {record_rows, tile_m, by_column, octets, (outputs + quads - 1) / quads};
    const long long blocks = warps ? (rows + kCombineThreads / 32 - 1) / (kCombineThreads / 32) : rows * c.parts;
    const dim3 grid((unsigned)std::max<long long>(1, std::min<long long>(blocks, (warps ? 3ll : 8ll) * sm_count)));
    switch (a.type) {
    case SATORI_F32: return launch_combine_type<SATORI_F32>(a, c, slices, grid, stream);
    case SATORI_F16: return launch_combine_type<SATORI_F16>(a, c, slices, grid, stream);
    default: return launch_combine_type<SATORI_BF16>(a, c, slices, grid, stream);
    }
}

extern "C" int satori_batch_create(satori_pages *pages, int q_heads, double rope_base, int rotary, satori_batch **out)
{
    return guarded([&]() -> int {
        if (!out) return set_error(SATORI_ERR_ARGUMENT, "out is null");
        if (!pages || pages->disposed) return set_error(SATORI_ERR_DISPOSED, "paged cache is disposed");
        if (q_heads <= 0 || q_heads % pages->kv_heads)
            return set_error(SATORI_ERR_ARGUMENT, "q_heads must be a positive multiple of kv_heads");
        if (rope_base != 0 && (!(rope_base > 0) || isinf(rope_base)))
            return set_error(SATORI_ERR_ARGUMENT, "rope_base must be 0 (no rotation) or positive and finite");
        if (rope_base != 0 && rotary == 0) rotary = pages->head_dim;
        if (rotary < 0 || rotary > pages->head_dim || rotary % 8)
            return set_error(SATORI_ERR_ARGUMENT, "rotary must be a multiple of 8, at most head_dim");
        satori_batch *b = new satori_batch();
        b->pages = pages;
        b->q_heads = q_heads;
        b->rope_base = rope_base;
        b->rotary = rope_base != 0 ? rotary : 0;
        b->shape.page_tokens = pages->tables.page_tokens();
        b->shape.kv_heads = pages->kv_heads;
        b->shape.group = q_heads / pages->kv_heads;
        const int sms = pages->ctx ? pages->ctx->sm_count : 148;
        if (on_tensor_cores(b))
            tensor_plan_shape(sms, b->shape);
        else if (on_f32_tiles(b))
            f32_plan_shape(pages->head_dim, sms, b->shape);
        else
            wide_plan_shape(sms, b->shape);
        ++pages->users;
        *out = b;
        return SATORI_OK;
    });
}

extern "C" int satori_batch_step(satori_batch *b, int n, const int *seqs, const int *counts)
{
    return guarded([&]() -> int {
        int rc = check_batch(b);
        if (rc) return rc;
        satori_pages *p = b->pages;
        if (p->ctx) {
            cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
            cudaError_t e = cudaStreamIsCapturing(p->ctx->stream, &status);
            if (e != cudaSuccess) return cuda_fail(e, "cudaStreamIsCapturing");
            if (status != cudaStreamCaptureStatusNone)
                return set_error(SATORI_ERR_NOT_SUPPORTED, "a step cannot be planned inside a stream capture");
        }
        if (n > 0 && !counts) return set_error(SATORI_ERR_ARGUMENT, "counts is null");
        long long rows = 0;
        for (int i = 0; i < n; ++i) rows += counts[i] > 0 ? counts[i] : 0;
        if (rows * b->q_heads > 0x7fffffff) return set_error(SATORI_ERR_NOT_SUPPORTED, "the step has too many rows");
        std::vector<PlanMember> members((size_t)std::max(n, 0));
        std::vector<satori_batch::Member> ids;
        ids.reserve(members.size());
        rc = pages_extend(p, n, seqs, counts);
        if (rc) return rc;                           // the last step's plan still stands
        b->planned = false;
        try {
            for (int i = 0; i < n; ++i) {
                const PageSequence &s = *p->tables.find(seqs[i]);
                members[i] = {s.pages.data(), (int)s.pages.size(), s.length, counts[i]};
                ids.push_back({seqs[i], s.version});
            }
            make_plan(b->shape, members, b->plan);
            if (p->ctx) rc = upload_plan(b);
        } catch (...) {
            pages_shrink(p, n, seqs, counts);
            throw;
        }
        if (rc) {
            pages_shrink(p, n, seqs, counts);
            return rc;
        }
        b->members.swap(ids);
        b->planned = true;
        return SATORI_OK;
    });
}

extern "C" int satori_batch_info(const satori_batch *batch, int *rows, int *segments, int *items, int *reallocations)
{
    satori_batch *b = const_cast<satori_batch *>(batch);
    int rc = check_batch(b);
    if (rc) return rc;
    if (rows) *rows = b->planned ? b->plan.head.rows : 0;
    if (segments) *segments = b->planned ? b->plan.head.segments : 0;
    if (items) *items = b->planned ? b->plan.head.items : 0;
    if (reallocations) *reallocations = b->reallocations;
    return SATORI_OK;
}

extern "C" int satori_batch_append_device(satori_batch *b, int layer, int in_type, const void *q, long long ldq,
                                          const void *k, long long ldk, const void *v, long long ldv, void *q_out)
{
    int rc = check_planned(b);
    if (rc) return rc;
    satori_pages *p = b->pages;
    if (layer < 0 || layer >= p->layers) return set_error(SATORI_ERR_ARGUMENT, "layer %d out of range", layer);
    if (in_type != SATORI_F32 && in_type != p->type)
        return set_error(SATORI_ERR_ARGUMENT, "inputs must be float32 or of the cache's type");
    if (b->plan.head.rows == 0) return SATORI_OK;
    if (!k || !v || (q && !q_out)) return set_error(SATORI_ERR_ARGUMENT, "null argument");
    const long long qw = (long long)b->q_heads * p->head_dim, kvw = (long long)p->kv_heads * p->head_dim;
    if (!ldq) ldq = qw;
    if (!ldk) ldk = kvw;
    if (!ldv) ldv = kvw;
    if ((q && ldq < qw) || ldk < kvw || ldv < kvw) return set_error(SATORI_ERR_ARGUMENT, "row stride below the row's length");
    const size_t es = type_size(in_type), os = type_size(p->type);
    if ((uintptr_t)k % es || (uintptr_t)v % es || (uintptr_t)q % es || (uintptr_t)q_out % os)
        return set_error(SATORI_ERR_ARGUMENT, "misaligned pointer");
    const long long n = b->plan.head.rows;
    if (q && ((rows_overlap(q_out, qw * os, qw * os, q, ldq * es, qw * es, n) && !(q_out == q && ldq == qw && in_type == p->type)) ||
              rows_overlap(q_out, qw * os, qw * os, k, ldk * es, kvw * es, n) || rows_overlap(q_out, qw * os, qw * os, v, ldv * es, kvw * es, n)))
        return set_error(SATORI_ERR_ARGUMENT, "q_out must not overlap an input (or be the packed q itself)");
    DeviceScope scope(p->ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    AppendArgs a = {};
    a.plan = reinterpret_cast<const DevPlan *>(b->d_plan);
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.q_out = q_out;
    a.pool = p->memory + (size_t)layer * p->layer_bytes();
    a.q_heads = b->q_heads;
    a.kv_heads = p->kv_heads;
    a.head_dim = p->head_dim;
    a.rotary = b->rotary;
    a.page_tokens = p->tables.page_tokens();
    const uintptr_t in = (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)(ldk * es) | (uintptr_t)(ldv * es) |
                         (uintptr_t)(q ? ldq * es : 0);
    const int wide_in = in % (4 * es) == 0, wide_out = (uintptr_t)q_out % (4 * os) == 0;
    const int rows = b->plan.head.rows, sms = p->ctx->sm_count;
    cudaStream_t st = p->ctx->stream;
    cudaError_t e;
    if (p->type == SATORI_F32)
        e = launch_append<SATORI_F32, SATORI_F32>(a, rows, wide_in, wide_out, sms, st);
    else if (p->type == SATORI_F16)
        e = in_type == SATORI_F32 ? launch_append<SATORI_F32, SATORI_F16>(a, rows, wide_in, wide_out, sms, st)
                                  : launch_append<SATORI_F16, SATORI_F16>(a, rows, wide_in, wide_out, sms, st);
    else
        e = in_type == SATORI_F32 ? launch_append<SATORI_F32, SATORI_BF16>(a, rows, wide_in, wide_out, sms, st)
                                  : launch_append<SATORI_BF16, SATORI_BF16>(a, rows, wide_in, wide_out, sms, st);
    return e == cudaSuccess ? SATORI_OK : cuda_fail(e, "append");
}

extern "C" int satori_batch_attention_device(satori_batch *b, int layer, const void *q, long long ldq, void *out,
                                             long long ldo, int out_type)
{
    int rc = check_planned(b);
    if (rc) return rc;
    satori_pages *p = b->pages;
    if (layer < 0 || layer >= p->layers) return set_error(SATORI_ERR_ARGUMENT, "layer %d out of range", layer);
    if (out_type != SATORI_F32 && out_type != p->type)
        return set_error(SATORI_ERR_ARGUMENT, "outputs must be float32 or of the cache's type");
    if (b->plan.head.rows == 0) return SATORI_OK;
    if (!q || !out) return set_error(SATORI_ERR_ARGUMENT, "null argument");
    const long long qw = (long long)b->q_heads * p->head_dim;
    if (!ldq) ldq = qw;
    if (!ldo) ldo = qw;
    if (ldq < qw || ldo < qw) return set_error(SATORI_ERR_ARGUMENT, "row stride below the row's length");
    if ((uintptr_t)q % type_size(p->type) || (uintptr_t)out % type_size(out_type))
        return set_error(SATORI_ERR_ARGUMENT, "misaligned pointer");
    const size_t es = type_size(p->type), os = type_size(out_type);
    if (rows_overlap(out, ldo * os, qw * os, q, ldq * es, qw * es, b->plan.head.rows))
        return set_error(SATORI_ERR_ARGUMENT, "out must not overlap q");
    DeviceScope scope(p->ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    const size_t rows = record_rows(b);
    BatchAttn a = {};
    a.plan = reinterpret_cast<const DevPlan *>(b->d_plan);
    a.pool = p->memory + (size_t)layer * p->layer_bytes();
    a.page_tokens = p->tables.page_tokens();
    a.kv_heads = p->kv_heads;
    a.group = b->shape.group;
    a.head_dim = p->head_dim;
    a.type = p->type;
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.out_f32 = out_type == SATORI_F32;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)p->head_dim));
    a.ctas = b->shape.ctas;
    a.err = p->ctx->d_err;
    const int layer_block = layer * p->tables.pages() * 2 * p->kv_heads;
    cudaError_t e = on_tensor_cores(b) ? launch_tensor_attention(a, p->map, layer_block, p->ctx->stream)
                    : on_f32_tiles(b)  ? launch_f32_attention(a, p->map, layer_block, p->ctx->stream)
                                       : launch_wide_attention(a, p->ctx->stream);
    if (e == cudaSuccess)
        e = launch_combine(a, (int)rows, b->shape.tile_m, on_tensor_cores(b), b->plan.head.merges,
                           p->ctx->sm_count, p->ctx->stream);
    return e == cudaSuccess ? SATORI_OK : cuda_fail(e, "batch attention");
}

extern "C" int satori_batch_destroy(satori_batch *b)
{
    if (!b) return SATORI_OK;
    if (b->pages->ctx) {
        DeviceScope scope(b->pages->ctx->device);
        cudaStreamSynchronize(b->pages->ctx->stream);
        cudaFree(b->d_plan);
        cudaFree(b->d_partials);
        cudaFree(b->d_rope);
        for (void *old : b->outgrown) cudaFree(old);
        b->staging.release();
    }
    pages_unref(b->pages);
    delete b;
    return SATORI_OK;
}
