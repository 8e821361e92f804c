// adapters.cu -- low-rank adapters of many requests beside a shared projection:
// out[p] = base[p] + scale_s * B_s (A_s x[p]), s the adapter slot of row p.
//
// The reference has no adapters; a host that serves fine-tuned variants of one model decodes their rows in one
// batch, the quantized projection once for all rows (satori_matrix_execute_device) and each row's own
// low-rank term beside it.
//
// One launch.  The rows are grouped by slot into items of up to 16, 32 or 64 rows; a thread-block cluster takes
// an item: its warps split the columns for t = A x, the partial t meet in shared memory and, across the
// cluster's CTAs, in distributed shared memory, and the warps split the output rows for B t.  So t never
// leaves the SMs, x is read once, base and out are touched once, and nothing is added by atomics: the order
// of every sum is fixed by the shapes.
//
// Both products run on the tensor cores at FP32 accuracy: x and t are cut into three bf16 parts each (24
// bits), a weight into as many as it needs to be exact (bf16 1, fp32 3), and the products of parts
// above 2^-24 of the whole are added in FP32 (3 and 6 MMAs per step).  Beside fp16 weights a row of t, or 32 columns
// of a row of x, is scaled by a power of two into fp16's range and cut into two fp16 parts (22 bits, or 2^-39 of the
// largest of them), which meet the weights as they are: 2 MMAs and no conversions.  Bytes bound it: the weights
// of the slots in use, x, base and out.  While outputs are written they move at 5.1 TB/s for 4000 rows of 3 slots (rank
// 64, 1536 -> 8960 in bf16, 56 of 97 us) and at 4.2 TB/s for 128 rows of 32 slots (3584 -> 18944 in fp16, 72 MB in 17 of
// 38 us).  Before that come the first product (the parts of x and of the weights) and the chain of loads, barriers and
// remote reads around it.  B streams through a ring of each warp's own in shared memory, filled by bulk copies a run or
// more ahead: a run's weights are contiguous, and the loads' latency was what the warps waited for.
#include "batch.cuh"
#include "common.cuh"
#include "paged_internal.h"
#include "staging.h"

#include <cooperative_groups.h>
#include <string.h>

#include <algorithm>
#include <array>
#include <climits>

using namespace satori;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kMaxRank = 128, kMaxCluster = 8, kItemRows = 64;
constexpr size_t kPlanInts = 1 << 14;          // of a row plan's first block

struct SlotDesc {
    const uint8_t *a, *b;                      // A [rank16][cols32] and B [rows][rank16], zero padded
    int rank16;                                // rank rounded up to 16; 0: no adapter
    float scale;
};

struct RowItem {
    int slot, row_off, rows;
};

// Header of a row plan, at an address that never changes, so that captured applications read the current
// assignment whatever its size.
struct DevRows {
    const RowItem *list;
    const int *rows;
    int items, pad[3];
};

struct AdapterArgs {
    const DevRows *plan;
    const SlotDesc *slots;
    const float *x, *base;
    float *out;
    long long ldx, ldbase, ldo;
    int n_slots;
    int splits;                                // clusters that share an item's outputs
    int rows, cols, cols32;                    // output rows, columns, columns rounded up to 32
    int wide_x, wide_out;                      // 16-byte accesses are possible
    unsigned *err;
};

// ------------------------------------------------------------------------------------------- bf16 parts
__device__ __forceinline__ uint32_t pack_bf16(float x, float y)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&b);
}

// (x, y) cut into N packed bf16 parts; each residual is exact in FP32.
template <int N>
__device__ __forceinline__ void split_values(float x, float y, uint32_t *part)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        part[i] = pack_bf16(x, y);
        x = __fsub_rn(x, __uint_as_float(part[i] << 16));
        y = __fsub_rn(y, __uint_as_float(part[i] & 0xFFFF0000u));
    }
}

template <int TYPE>
struct Weights;
template <>
struct Weights<SATORI_BF16> {
    static constexpr int kParts = 1, kBytes = 2;
};
template <>
struct Weights<SATORI_F16> {
    static constexpr int kParts = 1, kBytes = 2;
};
template <>
struct Weights<SATORI_F32> {
    static constexpr int kParts = 3, kBytes = 4;
};

// 4 consecutive weights as the B fragment of one MMA step: part[i][0] the first two, part[i][1] the others.
template <int TYPE>
__device__ __forceinline__ void weight_parts(const uint32_t *raw, uint32_t (*part)[2])
{
    if (TYPE != SATORI_F32) {
        part[0][0] = raw[0];
        part[0][1] = raw[1];
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t p[Weights<TYPE>::kParts];
            split_values<Weights<TYPE>::kParts>(__uint_as_float(raw[2 * h]), __uint_as_float(raw[2 * h + 1]), p);
#pragma unroll
            for (int i = 0; i < Weights<TYPE>::kParts; ++i) part[i][h] = p[i];
        }
    }
}

__device__ __forceinline__ void mma_bf16(float *d, const uint32_t *a, const uint32_t *b)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ void mma_f16(float *d, const uint32_t *a, const uint32_t *b)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// All products of parts i (of a, three) and j (of b) with i + j <= 2, small ones first.
template <int NB>
__device__ __forceinline__ void mma_parts(float *d, const uint32_t (*a)[4], const uint32_t (*b)[2])
{
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (j <= s) mma_bf16(d, a[s - j], b[j]);
}

// ------------------------------------------------------------------------------------------- the kernel
// RM: ranks at most.
template <int TYPE, int RM>
struct AdapterSmem {
    static constexpr int kRun = 32 * RM * Weights<TYPE>::kBytes;   // weights of 32 outputs at the largest rank
    static constexpr int kRing = kRun * (kRun <= 8192 ? 2 : 1);   // a warp's ring
    static constexpr int kSlots = 4;
    // t in parts, as the A fragments of the second product: [16 ranks][part][16 rows][lane].
    static constexpr int kParts = TYPE == SATORI_F16 ? 2 : 3;
    uint4 parts[RM / 16][kParts][kItemRows / 16][32];
    // FP32 t and the rows' scales, where the parts are made by each CTA for itself.
    float whole[TYPE == SATORI_F16 ? kItemRows : 1][RM + 4], unscale[kItemRows];
    union {
        struct {
            float red[kWarps][16][RM + 4];     // the warps' partial t of a 16-row tile
            float t[kItemRows][RM + 4];        // the CTA's partial t, read by the whole cluster
        };
        alignas(16) uint8_t ring[kWarps][kRing];
    };
    uint64_t full[kWarps][kSlots];
    int row[kItemRows];
};

// Where ranks r .. r + 3 (r a multiple of 4) of item row p lie in the fragments: the step of 16 ranks, and twice
// the lane plus the row's half.  In a whole run of 32 ranks lane q of a row holds 8 consecutive ones, 4 for
// each of two steps; in a last run of 16 it holds 4.
__device__ __forceinline__ void fragment_place(int rank, int p, int r, int &step, int &at)
{
    const int run = r / 32, in = r % 32;
    const bool both = 32 * run + 32 <= rank;
    step = 2 * run + (both ? in / 4 % 2 : 0);
    at = 2 * (p % 8 * 4 + (both ? in / 8 : in / 4)) + p / 8 % 2;
}

// The sum over the cluster of four values at the same place in every CTA.  (A call: in line its eight loads in flight
// took registers that the products then spilled.)
__device__ __noinline__ float4 cluster_sum(float *at, int ctas)
{
    cg::cluster_group cluster = cg::this_cluster();
    float4 v[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) v[c] = c < ctas ? *reinterpret_cast<const float4 *>(cluster.map_shared_rank(at, c)) : make_float4(0, 0, 0, 0);
    float4 sum = v[0];
#pragma unroll
    for (int c = 1; c < kMaxCluster; ++c) {
        sum.x += v[c].x;
        sum.y += v[c].y;
        sum.z += v[c].z;
        sum.w += v[c].w;
    }
    return sum;
}

template <int TYPE, int RM>
__global__ void __launch_bounds__(kThreads, sizeof(AdapterSmem<TYPE, RM>) <= 113 * 1024 ? 2 : 1) adapter_kernel(const AdapterArgs a)
{
    typedef Weights<TYPE> W;
    typedef AdapterSmem<TYPE, RM> Smem;
    // Tiles of 8 ranks taken together: their weights and sums fit the registers beside x.
    constexpr int NT = RM / 8 < (TYPE == SATORI_F32 ? 4 : 8) ? RM / 8 : (TYPE == SATORI_F32 ? 4 : 8);
    constexpr int RAW = W::kBytes * 8 / 4;     // words of 8 weights
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    pdl_launch_dependents();
    if (tid < kWarps * Smem::kSlots) mbar_init(&sm.full[tid / Smem::kSlots][tid % Smem::kSlots], 1);
    if (tid == 0) fence_mbar_init();
    uint32_t parity = 0;                       // bit s: this warp's slot s
    // The plan lay there when the launch before this one started: a copy on the stream brought it, and no launch
    // behind a copy starts before it.
    const int items = a.plan->items;
    const RowItem *list = a.plan->list;
    const int *rows = a.plan->rows;

    for (int unit = blockIdx.x / ctas; unit < items * a.splits; unit += gridDim.x / ctas) {
        const RowItem item = list[unit / a.splits];
        const int split = unit % a.splits;     // its share of the outputs; t is every share's own
        SlotDesc slot = {};
        // (A replay may follow an assignment of slots that these adapters lack: such rows get their base.)
        if (item.slot >= 0 && item.slot < a.n_slots)
            slot = a.slots[item.slot];
        else if (item.slot >= 0 && tid == 0)
            atomicOr(a.err, kDevErrSlot);
        const int rank = slot.rank16, tiles = (item.rows + 15) / 16;
        pdl_wait();
        __syncthreads();                       // the item before is done with the rows and the ring
        if (tid < kItemRows) sm.row[tid] = tid < item.rows ? rows[item.row_off + tid] : -1;
        __syncthreads();
        if (rank > 0) {
            // t = A x, 8 NT ranks at a time.  The warps are dealt to the item's tiles of 16 rows (1, 2 or 4 shares),
            // and those of a tile, over the cluster, take its runs of 32 columns in turn.  A lane holds 8 consecutive
            // columns of a row: the MMA's k index is a permutation of the run's columns, the same for x and A.
            const int shares = tiles > 2 ? 4 : tiles, per_tile = kWarps / shares, i = warp % shares;
            if (i < tiles) {
                const int row0 = sm.row[i * 16 + g], row1 = sm.row[i * 16 + 8 + g];
                for (int j0 = 0; j0 * 8 < rank; j0 += NT) {
                    const int nt = min(NT, rank / 8 - j0);
                    float acc[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = 0;
                    for (int k0 = (cta * per_tile + warp / shares) * 32; k0 < a.cols32; k0 += ctas * per_tile * 32) {
                        const int k = k0 + q * 8;
                        uint32_t raw[NT][RAW];
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            if (j < nt) {
                                const uint4 *src = reinterpret_cast<const uint4 *>(
                                    slot.a + ((long long)((j0 + j) * 8 + g) * a.cols32 + k) * W::kBytes);
#pragma unroll
                                for (int e = 0; e < RAW / 4; ++e) *reinterpret_cast<uint4 *>(&raw[j][4 * e]) = __ldg(src + e);
                            }
                        float x[2][8];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = h ? row1 : row0;
                            const float *src = a.x + row * a.ldx + k;
                            if (row >= 0 && a.wide_x && k + 8 <= a.cols) {
#pragma unroll
                                for (int e = 0; e < 8; e += 4) {
                                    const float4 v = __ldg(reinterpret_cast<const float4 *>(src + e));
                                    x[h][e] = v.x;
                                    x[h][e + 1] = v.y;
                                    x[h][e + 2] = v.z;
                                    x[h][e + 3] = v.w;
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e) x[h][e] = row >= 0 && k + e < a.cols ? __ldg(src + e) : 0.0f;
                            }
                        }
                        if (TYPE == SATORI_F16) {
                            // The run's columns of a row, scaled by a power of two, in two fp16 parts.
                            uint32_t xa[2][2][4];
                            float back[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float top = fabsf(x[h][0]);
#pragma unroll
                                for (int e = 1; e < 8; ++e) top = fmaxf(top, fabsf(x[h][e]));
                                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                                const int up = min(14 - ((int)(__float_as_uint(top) >> 23) - 127), 126);
                                const float scale = __uint_as_float((uint32_t)(127 + up) << 23);
                                back[h] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
                                for (int s = 0; s < 2; ++s)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const float a0 = x[h][4 * s + 2 * e] * scale, a1 = x[h][4 * s + 2 * e + 1] * scale;
                                        const __half2 hi = __floats2half2_rn(a0, a1);
                                        const float2 f = __half22float2(hi);
                                        const __half2 lo = __floats2half2_rn(a0 - f.x, a1 - f.y);
                                        xa[s][0][2 * e + h] = *reinterpret_cast<const uint32_t *>(&hi);
                                        xa[s][1][2 * e + h] = *reinterpret_cast<const uint32_t *>(&lo);
                                    }
                            }
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                if (j < nt) {
                                    float part[4] = {0, 0, 0, 0};
#pragma unroll
                                    for (int s = 0; s < 2; ++s) {
                                        mma_f16(part, xa[s][1], &raw[j][s * RAW / 2]);
                                        mma_f16(part, xa[s][0], &raw[j][s * RAW / 2]);
                                    }
#pragma unroll
                                    for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(part[e], back[e / 2], acc[j][e]);
                                }
                        } else {
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                uint32_t xa[3][4];
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        uint32_t p[3];
                                        split_values<3>(x[h][4 * s + 2 * e], x[h][4 * s + 2 * e + 1], p);
#pragma unroll
                                        for (int c = 0; c < 3; ++c) xa[c][2 * e + h] = p[c];
                                    }
#pragma unroll
                                for (int j = 0; j < NT; ++j)
                                    if (j < nt) {
                                        uint32_t wb[W::kParts][2];
                                        weight_parts<TYPE>(&raw[j][s * RAW / 2], wb);
                                        mma_parts<W::kParts>(acc[j], xa, wb);
                                    }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if (j < nt) {
                            float *d = &sm.red[warp][g][(j0 + j) * 8 + 2 * q];
                            *reinterpret_cast<float2 *>(d) = make_float2(acc[j][0], acc[j][1]);
                            *reinterpret_cast<float2 *>(d + 8 * (RM + 4)) = make_float2(acc[j][2], acc[j][3]);
                        }
                }
            }
            __syncthreads();
            for (int e = tid; e < item.rows * (rank / 4); e += kThreads) {
                const int p = e / (rank / 4), r = 4 * (e % (rank / 4));
                float4 sum = make_float4(0, 0, 0, 0);
                for (int w = p / 16; w < kWarps; w += shares) {
                    const float4 v = *reinterpret_cast<const float4 *>(&sm.red[w][p % 16][r]);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                *reinterpret_cast<float4 *>(&sm.t[p][r]) = sum;
            }
            cluster.sync();
            // Each CTA adds t over the cluster, scales it and cuts it into bf16 parts.  (Adding a share each and handing
            // the parts round took longer: 48 remote stores a value, one after the other.)  Rows behind the item's
            // keep what was there: so do the outputs nobody reads.
            for (int e = tid; e < item.rows * (rank / 4); e += kThreads) {
                const int p = e / (rank / 4), r = 4 * (e % (rank / 4));
                float4 sum = cluster_sum(&sm.t[p][r], ctas);
                sum.x *= slot.scale;
                sum.y *= slot.scale;
                sum.z *= slot.scale;
                sum.w *= slot.scale;
                if (TYPE == SATORI_F16) {
                    *reinterpret_cast<float4 *>(&sm.whole[p][r]) = sum;
                    continue;
                }
                uint32_t lo[3], hi[3];
                split_values<3>(sum.x, sum.y, lo);
                split_values<3>(sum.z, sum.w, hi);
                int step, at;
                fragment_place(rank, p, r, step, at);
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    uint32_t *to = reinterpret_cast<uint32_t *>(&sm.parts[step][k % Smem::kParts][p / 16][at >> 1]) + (at & 1);
                    to[0] = lo[k];
                    to[2] = hi[k];
                }
            }
            // From here on nobody reads another CTA's t, whose place the ring takes; and the parts are only written
            // again after the next item's first synchronisation, which every CTA of the cluster comes to.
            cluster.sync();
            if (TYPE == SATORI_F16) {
                // The power of two that brings a row's largest |t| into [2^14, 2^15), and its parts.
                for (int p = warp; p < tiles * 16; p += kWarps) {
                    float top = 0;
                    for (int r = lane; r < rank; r += 32) top = fmaxf(top, fabsf(sm.whole[p][r]));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                    int exponent = 0;
                    if (top > 0 && top < INFINITY) frexpf(top, &exponent);
                    const float scale = ldexpf(1.0f, min(15 - exponent, 126)), back = ldexpf(1.0f, max(exponent - 15, -126));
                    if (lane == 0) sm.unscale[p] = back;
                    for (int r = 4 * lane; r < rank; r += 128) {
                        const float4 v = *reinterpret_cast<const float4 *>(&sm.whole[p][r]);
                        int step, at;
                        fragment_place(rank, p, r, step, at);
                        float2 a0 = make_float2(v.x * scale, v.y * scale), a1 = make_float2(v.z * scale, v.w * scale);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const __half2 h0 = __floats2half2_rn(a0.x, a0.y), h1 = __floats2half2_rn(a1.x, a1.y);
                            uint32_t *to = reinterpret_cast<uint32_t *>(&sm.parts[step][k][p / 16][at >> 1]) + (at & 1);
                            to[0] = *reinterpret_cast<const uint32_t *>(&h0);
                            to[2] = *reinterpret_cast<const uint32_t *>(&h1);
                            const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                            a0 = make_float2(a0.x - f0.x, a0.y - f0.y);
                            a1 = make_float2(a1.x - f1.x, a1.y - f1.y);
                        }
                    }
                }
                __syncthreads();
            }
        }
        // out = base + B t: each warp takes runs of 32 output rows.  Lane (g, q) ends up with 8 consecutive
        // outputs, 8 q .. 8 q + 7, of tile rows g and g + 8: column 2 q + e of the MMA's n-tile j stands for
        // output 8 q + 2 j + e.  Ranks go 32 at a time (a lane holds 8 consecutive ones), the last 16 of an odd
        // number of 16s with 4 a lane.
        constexpr int C32 = 1;                 // runs of 32 ranks held at once
        const int run_bytes = 32 * rank * W::kBytes, slots = rank ? min(Smem::kSlots, Smem::kRing / run_bytes) : 1;
        const int runs = (a.rows + 31) / 32, stride = a.splits * ctas * kWarps, first = (split * ctas + cta) * kWarps + warp;
        auto fetch = [&](int run, int s) {
            const int bytes = min(32, a.rows - run * 32) * rank * W::kBytes;
            mbar_expect_tx(&sm.full[warp][s], (uint32_t)bytes);
            bulk_g2s(&sm.ring[warp][s * run_bytes], slot.b + (long long)run * run_bytes, (uint32_t)bytes, &sm.full[warp][s]);
        };
        if (rank > 0 && lane == 0) {
            // The ring's memory was last touched by ordinary accesses.
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (int s = 0; s < slots; ++s)
                if (first + s * stride < runs) fetch(first + s * stride, s);
        }
        int s = 0;
        for (int run = first; run < runs; run += stride, s = s + 1 == slots ? 0 : s + 1) {
            const int o0 = run * 32, o = o0 + 8 * q;
            const uint8_t *weights = &sm.ring[warp][s * run_bytes];
            bool arrived = rank == 0;
            for (int i = 0; i < tiles; ++i) {
                float base[2][8], acc[4][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = sm.row[i * 16 + h * 8 + g];
                    const float *src = a.base + row * a.ldbase + o;
                    if (row >= 0 && a.wide_out && o + 8 <= a.rows) {
                        *reinterpret_cast<float4 *>(&base[h][0]) = *reinterpret_cast<const float4 *>(src);
                        *reinterpret_cast<float4 *>(&base[h][4]) = *reinterpret_cast<const float4 *>(src + 4);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) base[h][e] = row >= 0 && o + e < a.rows ? src[e] : 0.0f;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] = 0;
                if (!arrived && !mbar_wait_bounded(&sm.full[warp][s], parity >> s & 1u)) atomicOr(a.err, kDevErrTimeout);
                for (int r0 = 0; r0 < rank; r0 += 32 * C32) {
                    uint32_t raw[C32][4][RAW];
#pragma unroll
                        for (int c = 0; c < C32; ++c)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                // (Rows behind the last output hold an earlier run's weights; their sums are not stored.)
                                const int r = r0 + 32 * c;
                                const uint8_t *src = weights + ((8 * (g >> 1) + 2 * j + (g & 1)) * rank + r) * W::kBytes;
                                if (r + 32 <= rank) {
                                    const uint4 *from = reinterpret_cast<const uint4 *>(src + q * 8 * W::kBytes);
#pragma unroll
                                    for (int e = 0; e < RAW / 4; ++e) *reinterpret_cast<uint4 *>(&raw[c][j][4 * e]) = from[e];
                                } else if (r < rank) {
                                    const uint2 *from = reinterpret_cast<const uint2 *>(src + q * 4 * W::kBytes);
#pragma unroll
                                    for (int e = 0; e < RAW / 4; ++e) *reinterpret_cast<uint2 *>(&raw[c][j][2 * e]) = from[e];
                                }
                            }
#pragma unroll
                    for (int c = 0; c < C32; ++c)
#pragma unroll
                        for (int step = 0; step < 2; ++step) {
                            const int r = r0 + 32 * c + 16 * step;
                            if (r >= rank) continue;
                            uint32_t frag[Smem::kParts][4];
#pragma unroll
                            for (int p = 0; p < Smem::kParts; ++p)
                                *reinterpret_cast<uint4 *>(frag[p]) = sm.parts[r / 16][p][i][lane];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t *words = &raw[c][j][step * RAW / 2];
                                if (TYPE == SATORI_F16) {
                                    mma_f16(acc[j], frag[1], words);
                                    mma_f16(acc[j], frag[0], words);
                                } else {
                                    uint32_t wb[W::kParts][2];
                                    weight_parts<TYPE>(words, wb);
                                    mma_parts<W::kParts>(acc[j], frag, wb);
                                }
                            }
                        }
                }
                if (!arrived) {
                    parity ^= 1u << s;
                    arrived = true;
                }
                if (TYPE == SATORI_F16 && rank > 0)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float back = sm.unscale[i * 16 + (e >> 1) * 8 + g];
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j][e] *= back;
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = sm.row[i * 16 + h * 8 + g];
                    if (row < 0) continue;
                    float *out = a.out + row * a.ldo + o;
                    if (a.wide_out && o + 8 <= a.rows) {
#pragma unroll
                        for (int j = 0; j < 4; j += 2)
                            *reinterpret_cast<float4 *>(out + 2 * j) =
                                make_float4(base[h][2 * j] + acc[j][2 * h], base[h][2 * j + 1] + acc[j][2 * h + 1],
                                            base[h][2 * j + 2] + acc[j + 1][2 * h], base[h][2 * j + 3] + acc[j + 1][2 * h + 1]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (o + e < a.rows) out[e] = base[h][e] + acc[e / 2][2 * h + (e & 1)];
                    }
                }
            }
            if (rank > 0) {
                __syncwarp();                  // the warp has read the slot
                if (lane == 0 && run + slots * stride < runs) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    fetch(run + slots * stride, s);
                }
            }
        }
    }
    pdl_wait();                // also without an item: launches behind this one count on the end of those before
}

}  // namespace

struct satori_adapters {
    satori_ctx *ctx = nullptr;
    int rows = 0, cols = 0, slots = 0, max_rank = 0, max_rank16 = 0, type = 0;
    uint8_t *d_weights = nullptr;
    SlotDesc *d_slots = nullptr;
    size_t a_bytes() const { return (size_t)max_rank16 * cols32() * type_size(type); }
    size_t b_bytes() const { return ((size_t)rows * max_rank16 * type_size(type) + 255) / 256 * 256; }
    int cols32() const { return (cols + 31) / 32 * 32; }
};

struct satori_adapter_rows {
    satori_ctx *ctx = nullptr;
    int rows = -1, top_slot = -1;              // rows assigned, highest slot used
    int items = 0;
    int *d_plan = nullptr;                     // kPlanInts: the header, and the lists behind it where they fit
    int *d_lists = nullptr;                    // longer lists
    size_t list_ints = 0;
    std::vector<void *> outgrown;              // may still be read by launches that are queued
    Staging staging;
};

namespace {

// A captured change of the weights or slots would be repeated by every replay.
int check_not_capturing(const satori_ctx *ctx, const char *what)
{
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(ctx->stream, &status);
    if (e != cudaSuccess) return cuda_fail(e, "cudaStreamIsCapturing");
    if (status != cudaStreamCaptureStatusNone) return set_error(SATORI_ERR_NOT_SUPPORTED, "%s inside a stream capture", what);
    return SATORI_OK;
}

// How many clusters of each size up to 8 run at once.  The SMs of a GPC hold whole clusters, so it's less than the
// CTAs' number divided by the cluster's.
template <typename Kernel>
std::array<int, kMaxCluster + 1> resident_clusters(Kernel kernel, size_t smem, int sm_count)
{
    std::array<int, kMaxCluster + 1> got = {};
    for (int size = 1; size <= kMaxCluster; ++size) {
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)size;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(sm_count * 8 * size));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&got[size], kernel, &cfg) != cudaSuccess || got[size] < 1) {
            cudaGetLastError();
            got[size] = std::max(1, sm_count / size);
        }
    }
    return got;
}

template <int TYPE, int RM>
cudaError_t launch_variant(AdapterArgs a, int items, int sm_count, cudaStream_t stream)
{
    auto kernel = adapter_kernel<TYPE, RM>;
    const size_t smem = sizeof(AdapterSmem<TYPE, RM>);
    cudaError_t e = opt_in_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    // All items are resident at once where that can be: a second wave costs as much as the first (2400 rows of one
    // slot, rank 64, 8960 outputs, in 38 items: 97 us on clusters of 4, 73 on 6).  An item may have several clusters, of which all
    // compute t and each writes a share of the outputs.  Of the clusters' sizes that fit, the one whose warps have
    // the fewest runs of 32, of columns for t and (twice the work) of outputs, in turn: one slot's 22 rows, rank 64,
    // 8960 outputs in FP32 take 13 us, with one cluster an item 28.8.
    static const std::array<int, kMaxCluster + 1> resident = resident_clusters(kernel, smem, sm_count);
    const int column_runs = a.cols32 / 32, runs = (a.rows + 31) / 32;
    auto turns = [](int n, int among) { return (n + among - 1) / among; };
    int cluster = 1, least = INT_MAX;
    a.splits = 1;
    for (int size = kMaxCluster; size >= 1; --size) {
        if (items > resident[size]) continue;
        const int most = resident[size] / items, each = turns(runs, size * kWarps * most);
        const int cost = turns(column_runs, size * kWarps) + 2 * each;
        if (cost < least) {
            least = cost;
            cluster = size;
            a.splits = turns(runs, size * kWarps * each);
        }
    }
    const int clusters = std::max(1, std::min(items * a.splits, 8 * sm_count / cluster));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int TYPE>
cudaError_t launch_adapters(const AdapterArgs &a, int rank, int items, int sm_count, cudaStream_t stream)
{
    if (rank <= 16) return launch_variant<TYPE, 16>(a, items, sm_count, stream);
    if (rank <= 32) return launch_variant<TYPE, 32>(a, items, sm_count, stream);
    if (rank <= 64) return launch_variant<TYPE, 64>(a, items, sm_count, stream);
    return launch_variant<TYPE, 128>(a, items, sm_count, stream);
}

}  // namespace

extern "C" int satori_adapters_create(satori_ctx *ctx, int rows, int cols, int slots, int max_rank, int type,
                                      satori_adapters **out)
{
    return guarded([&]() -> int {
        if (!ctx || !out) return set_error(SATORI_ERR_ARGUMENT, "ctx/out is null");
        if (rows <= 0 || cols <= 0 || slots <= 0 || max_rank <= 0)
            return set_error(SATORI_ERR_ARGUMENT, "rows/cols/slots/max_rank must be positive");
        if (rows > (1 << 24) || cols > (1 << 24)) return set_error(SATORI_ERR_NOT_SUPPORTED, "more than 2^24 rows or columns");
        if (max_rank > kMaxRank) return set_error(SATORI_ERR_NOT_SUPPORTED, "ranks above %d are not supported", kMaxRank);
        if (!type_size(type)) return set_error(SATORI_ERR_ARGUMENT, "unsupported type %d", type);
        DeviceScope scope(ctx->device);
        if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
        int rc = check_not_capturing(ctx, "adapters cannot be created");
        if (rc) return rc;
        satori_adapters *s = new satori_adapters();
        s->ctx = ctx;
        s->rows = rows;
        s->cols = cols;
        s->slots = slots;
        s->max_rank = max_rank;
        s->max_rank16 = (max_rank + 15) / 16 * 16;
        s->type = type;
        cudaError_t e = cudaMalloc(&s->d_weights, (s->a_bytes() + s->b_bytes()) * (size_t)slots);
        if (e == cudaSuccess) e = cudaMalloc(&s->d_slots, sizeof(SlotDesc) * (size_t)slots);
        if (e == cudaSuccess) e = cudaMemsetAsync(s->d_slots, 0, sizeof(SlotDesc) * (size_t)slots, ctx->stream);
        if (e != cudaSuccess) {
            rc = cuda_fail(e, "allocate adapters");
            satori_adapters_destroy(s);
            return rc;
        }
        *out = s;
        return SATORI_OK;
    });
}

extern "C" int satori_adapters_load(satori_adapters *s, int slot, int rank, const void *a, long long lda, const void *b,
                                    long long ldb, float scale)
{
    if (!s) return set_error(SATORI_ERR_DISPOSED, "adapters are disposed");
    if (slot < 0 || slot >= s->slots) return set_error(SATORI_ERR_ARGUMENT, "slot %d out of range", slot);
    if (rank < 0 || rank > s->max_rank)
        return set_error(SATORI_ERR_ARGUMENT, "rank %d is outside 0..%d", rank, s->max_rank);
    if (rank > 0 && (!a || !b)) return set_error(SATORI_ERR_ARGUMENT, "null argument");
    if (!lda) lda = s->cols;
    if (!ldb) ldb = rank;
    if (rank > 0 && (lda < s->cols || ldb < rank)) return set_error(SATORI_ERR_ARGUMENT, "row stride below the row's length");
    if (!(scale - scale == 0)) return set_error(SATORI_ERR_ARGUMENT, "scale must be finite");
    satori_ctx *ctx = s->ctx;
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    int rc = check_not_capturing(ctx, "adapters cannot change");
    if (rc) return rc;
    const size_t es = type_size(s->type), ka = (size_t)s->cols32() * es;
    const int rank16 = (rank + 15) / 16 * 16;
    uint8_t *da = s->d_weights + (size_t)slot * s->a_bytes();
    uint8_t *db = s->d_weights + (size_t)s->slots * s->a_bytes() + (size_t)slot * s->b_bytes();
    SlotDesc d = {da, db, rank16, scale};
    cudaError_t e = cudaSuccess;
    if (rank > 0) {
        // Padding columns and ranks are zero, so whole tiles may be multiplied.
        e = cudaMemsetAsync(da, 0, s->a_bytes(), ctx->stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(db, 0, s->b_bytes(), ctx->stream);
        if (e == cudaSuccess)
            e = cudaMemcpy2DAsync(da, ka, a, (size_t)lda * es, (size_t)s->cols * es, (size_t)rank, cudaMemcpyDefault, ctx->stream);
        if (e == cudaSuccess)
            e = cudaMemcpy2DAsync(db, (size_t)rank16 * es, b, (size_t)ldb * es, (size_t)rank * es, (size_t)s->rows,
                                  cudaMemcpyDefault, ctx->stream);
    }
    if (e == cudaSuccess) e = cudaMemcpyAsync(s->d_slots + slot, &d, sizeof d, cudaMemcpyHostToDevice, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);      // the caller may reuse its memory
    return e == cudaSuccess ? SATORI_OK : cuda_fail(e, "load adapter");
}

extern "C" int satori_adapters_destroy(satori_adapters *s)
{
    if (!s) return SATORI_OK;
    DeviceScope scope(s->ctx->device);
    cudaStreamSynchronize(s->ctx->stream);
    cudaFree(s->d_weights);
    cudaFree(s->d_slots);
    delete s;
    return SATORI_OK;
}

extern "C" int satori_adapter_rows_create(satori_ctx *ctx, satori_adapter_rows **out)
{
    return guarded([&]() -> int {
        if (!ctx || !out) return set_error(SATORI_ERR_ARGUMENT, "ctx/out is null");
        satori_adapter_rows *r = new satori_adapter_rows();
        r->ctx = ctx;
        *out = r;
        return SATORI_OK;
    });
}

extern "C" int satori_adapter_rows_assign(satori_adapter_rows *r, int n, const int *slots)
{
    return guarded([&]() -> int {
        if (!r) return set_error(SATORI_ERR_DISPOSED, "adapter rows are disposed");
        if (n < 0 || (n > 0 && !slots)) return set_error(SATORI_ERR_ARGUMENT, "bad slot list");
        int top = -1;
        for (int i = 0; i < n; ++i) {
            if (slots[i] < -1) return set_error(SATORI_ERR_ARGUMENT, "slot %d is negative", slots[i]);
            top = std::max(top, slots[i]);
        }
        satori_ctx *ctx = r->ctx;
        DeviceScope scope(ctx->device);
        if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
        int rc = check_not_capturing(ctx, "rows cannot be assigned");
        if (rc) return rc;
        cudaError_t e = cudaSuccess;
        std::vector<int> order((size_t)n);
        for (int i = 0; i < n; ++i) order[i] = i;
        std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return slots[x] < slots[y]; });
        // The largest items (their rows share the weights' loads) whose clusters still give the SMs two CTAs each.
        std::vector<RowItem> items;
        for (int most = kItemRows; most >= 16; most /= 2) {
            items.clear();
            for (int i = 0; i < n;) {
                int end = i;
                while (end < n && slots[order[end]] == slots[order[i]]) ++end;
                for (int at = i; at < end; at += most) items.push_back({slots[order[i]], at, std::min(most, end - at)});
                i = end;
            }
            if ((int)items.size() * kMaxCluster >= 2 * ctx->sm_count) break;
        }
        const size_t head_ints = sizeof(DevRows) / 4, item_ints = items.size() * sizeof(RowItem) / 4, ints = item_ints + (size_t)n;
        const bool apart = head_ints + ints > kPlanInts;
        if (!r->d_plan && (e = cudaMalloc(&r->d_plan, kPlanInts * 4)) != cudaSuccess) return cuda_fail(e, "allocate adapter rows");
        if (apart && ints > r->list_ints) {
            const size_t count = std::max(ints, 2 * r->list_ints);
            int *fresh = nullptr;
            r->outgrown.reserve(r->outgrown.size() + 1);
            if ((e = cudaMalloc(&fresh, count * 4)) != cudaSuccess) return cuda_fail(e, "allocate adapter rows");
            if (r->d_lists) r->outgrown.push_back(r->d_lists);
            r->d_lists = fresh;
            r->list_ints = count;
        }
        void *buffer = nullptr;
        if ((e = r->staging.take((head_ints + ints) * 4, &buffer)) != cudaSuccess) return cuda_fail(e, "stage adapter rows");
        int *stage = static_cast<int *>(buffer);
        int *lists = apart ? r->d_lists : r->d_plan + head_ints;
        DevRows head = {};
        head.list = reinterpret_cast<const RowItem *>(lists);
        head.rows = lists + item_ints;
        head.items = (int)items.size();
        memcpy(stage, &head, sizeof head);
        if (n) memcpy(stage + head_ints, items.data(), item_ints * 4);
        if (n) memcpy(stage + head_ints + item_ints, order.data(), (size_t)n * 4);
        r->rows = -1;
        if (apart) e = cudaMemcpyAsync(lists, stage + head_ints, ints * 4, cudaMemcpyHostToDevice, ctx->stream);
        if (e == cudaSuccess) e = r->staging.send(r->d_plan, (apart ? head_ints : head_ints + ints) * 4, ctx->stream);
        if (e != cudaSuccess) return cuda_fail(e, "upload adapter rows");
        r->rows = n;
        r->top_slot = top;
        r->items = head.items;
        return SATORI_OK;
    });
}

extern "C" int satori_adapter_rows_destroy(satori_adapter_rows *r)
{
    if (!r) return SATORI_OK;
    DeviceScope scope(r->ctx->device);
    cudaStreamSynchronize(r->ctx->stream);
    cudaFree(r->d_plan);
    cudaFree(r->d_lists);
    for (void *old : r->outgrown) cudaFree(old);
    r->staging.release();
    delete r;
    return SATORI_OK;
}

extern "C" int satori_adapters_apply_device(satori_adapters *s, const satori_adapter_rows *r, const float *x, long long ldx,
                                            const float *base, long long ldbase, float *out, long long ldo)
{
    if (!s) return set_error(SATORI_ERR_DISPOSED, "adapters are disposed");
    if (!r) return set_error(SATORI_ERR_DISPOSED, "adapter rows are disposed");
    // The assignment was uploaded on its own context's stream: nothing orders it before this context's launch.
    if (r->ctx != s->ctx) return set_error(SATORI_ERR_ARGUMENT, "adapters and rows belong to different contexts");
    if (r->rows < 0) return set_error(SATORI_ERR_ARGUMENT, "no rows are assigned yet");
    if (r->top_slot >= s->slots)
        return set_error(SATORI_ERR_ARGUMENT, "slot %d is assigned; these adapters have %d", r->top_slot, s->slots);
    if (r->rows == 0) return SATORI_OK;
    if (!x || !base || !out) return set_error(SATORI_ERR_ARGUMENT, "null argument");
    if (!ldx) ldx = s->cols;
    if (!ldbase) ldbase = s->rows;
    if (!ldo) ldo = s->rows;
    if (ldx < s->cols || ldbase < s->rows || ldo < s->rows)
        return set_error(SATORI_ERR_ARGUMENT, "row stride below the row's length");
    if (((uintptr_t)x | (uintptr_t)base | (uintptr_t)out) % 4) return set_error(SATORI_ERR_ARGUMENT, "misaligned pointer");
    const long long width = s->rows * 4ll;
    if (rows_overlap(out, ldo * 4, width, x, ldx * 4, s->cols * 4ll, r->rows) ||
        (rows_overlap(out, ldo * 4, width, base, ldbase * 4, width, r->rows) && !(out == base && ldo == ldbase)))
        return set_error(SATORI_ERR_ARGUMENT, "output must not overlap input (or be base itself)");
    DeviceScope scope(s->ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    AdapterArgs a = {};
    a.plan = reinterpret_cast<const DevRows *>(r->d_plan);
    a.slots = s->d_slots;
    a.n_slots = s->slots;
    a.x = x;
    a.base = base;
    a.out = out;
    a.ldx = ldx;
    a.ldbase = ldbase;
    a.ldo = ldo;
    a.rows = s->rows;
    a.cols = s->cols;
    a.cols32 = s->cols32();
    a.wide_x = (uintptr_t)x % 16 == 0 && ldx % 4 == 0;
    a.wide_out = ((uintptr_t)base | (uintptr_t)out) % 16 == 0 && ldbase % 4 == 0 && ldo % 4 == 0;
    a.err = s->ctx->d_err;
    const int sms = s->ctx->sm_count;
    cudaError_t e;
    switch (s->type) {
    case SATORI_F32: e = launch_adapters<SATORI_F32>(a, s->max_rank16, r->items, sms, s->ctx->stream); break;
    case SATORI_F16: e = launch_adapters<SATORI_F16>(a, s->max_rank16, r->items, sms, s->ctx->stream); break;
    default: e = launch_adapters<SATORI_BF16>(a, s->max_rank16, r->items, sms, s->ctx->stream);
    }
    return e == cudaSuccess ? SATORI_OK : cuda_fail(e, "apply adapters");
}

extern "C" int satori_matrix_execute_adapted_device(satori_matrix *m, satori_adapters *s, const satori_adapter_rows *r,
                                                    const float *dx, float *dy, int order)
{
    if (!m) return set_error(SATORI_ERR_DISPOSED, "matrix is disposed");
    if (!s) return set_error(SATORI_ERR_DISPOSED, "adapters are disposed");
    if (!r) return set_error(SATORI_ERR_DISPOSED, "adapter rows are disposed");
    if (s->rows != m->rows || s->cols != m->cols)
        return set_error(SATORI_ERR_ARGUMENT, "adapters of %d x %d beside a %d x %d matrix", s->rows, s->cols, m->rows, m->cols);
    if (s->ctx != m->ctx) return set_error(SATORI_ERR_ARGUMENT, "adapters and matrix belong to different contexts");
    if (r->ctx != s->ctx) return set_error(SATORI_ERR_ARGUMENT, "adapters and rows belong to different contexts");
    if (r->rows < 0) return set_error(SATORI_ERR_ARGUMENT, "no rows are assigned yet");
    if (r->top_slot >= s->slots)
        return set_error(SATORI_ERR_ARGUMENT, "slot %d is assigned; these adapters have %d", r->top_slot, s->slots);
    if (r->rows == 0) return SATORI_OK;
    if (dx && dy && rows_overlap(dy, m->rows * 4ll, m->rows * 4ll, dx, m->cols * 4ll, m->cols * 4ll, r->rows))
        return set_error(SATORI_ERR_ARGUMENT, "output must not overlap input");
    DeviceScope scope(m->ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    int rc = satori_matrix_execute_device(m, dx, dy, r->rows, order);
    return rc ? rc : satori_adapters_apply_device(s, r, dx, 0, dy, 0, dy, 0);
}

