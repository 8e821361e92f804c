// batch_attn_f32.cu -- attention of a batch over a paged FP32 cache with heads of up to 128, on the FP32 units (the
// tensor cores would round its products).  HD below is 32, 64, 96 or 128: columns from the head's own size on are
// zeros (the copies of K and V fill them in) and are neither read from q nor written.
//
// The formulas are the FP32-unit kernel's for other caches (one pass over the keys, running maximum and sum);
// here the keys come through a ring of shared memory tiles, so that the loads of the next blocks run under the
// arithmetic of this one.  One CTA per SM works through its share of the plan's items; warp 8's elected thread
// loads each block of 64 keys as a K and a V tile (TMA, 32 columns of 128 bytes a row with the 128-byte swizzle:
// 8 threads that read 16 bytes of 8 consecutive rows, or of one row, meet 8 different bank groups), warps 0-7
// compute.  By the rows of the item's tile:
//  * at most 8 rows (the query heads of one KV head of one request): each warp takes 8 keys of every block on its
//    own, with a running maximum of its own and no barrier among warps.  A lane holds 4 columns of the queries
//    and of the outputs; the 64 partial dot products meet in a halving exchange (62 shuffles) that leaves each
//    lane one key and two rows.  HBM bounds it: 64 KB a block of 128-wide heads are 2800 clocks, its
//    instructions about 1700.
//  * up to 64, 96 or 128 rows (a shared prefix, a prompt): 4, 6 or 8 rows x 4 scores and x HD / 16 outputs per
//    thread.  A 16-byte read of shared memory takes a warp 4 clocks, or 2 where each half of it reads one address
//    (the queries, the weights), a packed product 2 clocks of one of four units: with 8 rows the products take
//    longer than the reads (256 : 256 clocks for 4 columns of the scores, 512 : 384 for 4 keys of the outputs),
//    with 4 rows the reads take longer, for half the work (192 : 128, 320 : 256).
// Products are packed two to an instruction, which halves the issue slots, not the arithmetic.
//
// Measured with heads of 128: one request of 300 tokens (28 heads over 4) 6.5 us, of 32768 tokens 35.6 us (20.8 at
// the rate of HBM), 16 requests of 4096 tokens 51 us (41.6 at the rate of HBM), 16 requests (12 heads over 2: 96
// rows) that share 8192 tokens 35 us and 65536 tokens 175 us, of which the packed products are 14 and 110 us.
#include "batch.cuh"
#include "common.cuh"

#include <algorithm>

namespace satori {

namespace {

constexpr int kWarps = 8, kCompute = kWarps * 32, kThreads = kCompute + 128;
constexpr int kTileM = 128, kBlock = 64, kFewRows = 8;
// The 65536 registers: 168 a thread at the launch, of which the loader's four warps hand most to the others.
constexpr int kLoaderRegs = 40, kComputeRegs = 232;
static_assert(128 * kLoaderRegs + kCompute * kComputeRegs <= kThreads * 168, "registers");

template <int HD>
struct Layout {
    static constexpr int kSub = kBlock * 128;                      // 64 rows of 32 columns
    static constexpr int kTile = kSub * (HD / 32);
    static constexpr int kStages = HD <= 64 ? 8 : HD <= 96 ? 6 : 4;
};

template <int HD>
struct alignas(1024) Smem {
    uint8_t stages[Layout<HD>::kStages][Layout<HD>::kTile];
    float q[kTileM * HD];                              // see q_chunk
    union {
        float p[kTileM * kBlock];                      // weights, see p_at
        float few[kWarps][kFewRows + 1][kFewRows];     // a warp's weights [key][row], then the rows' factors
    };
    float few_m[kWarps][kFewRows], few_l[kWarps][kFewRows];
    uint64_t full[Layout<HD>::kStages], empty[Layout<HD>::kStages];
    int limit[kTileM], row[kTileM], head[kTileM];      // visible keys of the segment, global row, query head
    volatile int abort;
};

__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// True in one lane of the converged warp (see the tensor-core kernel).
__device__ __forceinline__ bool elect_one()
{
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 r;\n\telect.sync r|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void load_3d(uint32_t dst, const void *map, int c0, int c1, int c2, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void load_4d(uint32_t dst, const void *map, int token, int block, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(token), "r"(0), "r"(block), "r"(smem_u32(bar)) : "memory");
}

template <int HD>
struct Ring {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next()
    {
        if (++stage == Layout<HD>::kStages) {
            stage = 0;
            parity ^= 1u;
        }
    }
};

__device__ __forceinline__ PlanItem load_item(const DevPlan *plan, int i)
{
    PlanItem item;
    const int4 *src = reinterpret_cast<const int4 *>(plan_array<PlanItem>(plan, plan->items) + i);
    int4 *dst = reinterpret_cast<int4 *>(&item);
#pragma unroll
    for (int k = 0; k < (int)(sizeof(PlanItem) / 16); ++k) dst[k] = __ldg(src + k);
    return item;
}

// 16-byte chunk c (4 columns) of row `key` of a tile.
__device__ __forceinline__ float4 tile_chunk(const uint8_t *tile, int key, int c)
{
    return *reinterpret_cast<const float4 *>(tile + (c >> 3) * (kBlock * 128) + key * 128 + (((c ^ key) & 7) << 4));
}

// Rows of the queries and of the weights change their order by RI rows, so that the two rows that a warp reads
// (RI apart) lie in different banks without padding.
template <int HD, int RI>
__device__ __forceinline__ int q_chunk(int row, int c) { return row * HD + (c ^ ((row / RI) & 1)) * 4; }
template <int RI>
__device__ __forceinline__ int p_at(int row, int key) { return row * kBlock + (key ^ (((row / RI) & 1) << 4)); }

__device__ __forceinline__ float2 lo2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

struct Args {
    BatchAttn a;
    int layer_block;
};

// The item's K and V tiles in turn.  PER: pages of a block; their numbers are fetched a block ahead.
template <int HD, int PER, typename Wait>
__device__ __forceinline__ bool load_tiles(const Args &t, const CUtensorMap &map, Smem<HD> &sm, const int *pages,
                                           const PlanItem &item, Ring<HD> &ring, int &units, Wait &wait)
{
    typedef Layout<HD> L;
    constexpr int kBox = kBlock / PER;
    const int shift = __ffs(t.a.page_tokens) - 1, mask = t.a.page_tokens - 1, page_blocks = 2 * t.a.kv_heads;
    auto fetch = [&](int j, int (&id)[PER]) {
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            const int key = (item.block0 + j) * kBlock + b * kBox;
            id[b] = key < item.keys ? __ldg(pages + (key >> shift)) : 0;
        }
    };
    int id[PER];
    fetch(0, id);
    for (int j = 0; j < item.blocks; ++j) {
        int next[PER];
        if (j + 1 < item.blocks) fetch(j + 1, next);
        const int key0 = (item.block0 + j) * kBlock, boxes = (min(kBlock, item.keys - key0) + kBox - 1) / kBox;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            uint64_t *full = &sm.full[ring.stage];
            if (!wait(&sm.empty[ring.stage], ring.parity ^ 1u)) return false;
            const uint32_t to = smem_u32(sm.stages[0]) + ring.stage * L::kTile;
            const int block0 = t.layer_block + kv * t.a.kv_heads + item.kv_head;
            mbar_expect_tx(full, (uint32_t)(boxes * kBox * HD * 4));
            if (PER == 1 && t.a.head_dim % 32 == 0) {
                load_4d(to, &map, key0 & mask, block0 + id[0] * page_blocks, full);
            } else {
#pragma unroll
                for (int b = 0; b < PER; ++b)
                    if (b < boxes)
#pragma unroll
                        for (int c = 0; c < HD / 32; ++c)
                            load_3d(to + c * L::kSub + b * kBox * 128, &map, c * 32, PER == 1 ? key0 & mask : 0,
                                    block0 + id[b] * page_blocks, full);
            }
            ring.next();
            ++units;
        }
        if (j + 1 < item.blocks)
#pragma unroll
            for (int b = 0; b < PER; ++b) id[b] = next[b];
    }
    return true;
}

__device__ __forceinline__ void store_out(const BatchAttn &a, int row, int head, int d, float v)
{
    reinterpret_cast<float *>(a.out)[(long long)row * a.ldo + (long long)head * a.head_dim + d] = v;
}

// Rows' indices and limits, and their queries times log2(e) / sqrt(d).
template <int HD, int RI>
__device__ __forceinline__ void load_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item, Smem<HD> &sm, int rows)
{
    const int tid = threadIdx.x;
    if (tid < rows) {
        const int m = item.m0 + tid;
        const bool live = tid < item.m;
        int2 own = make_int2(0, 0);
        if (live) own = __ldg(reinterpret_cast<const int2 *>(plan_array<PlanRow>(plan, plan->seg_rows) + item.row_off) + m / a.group);
        sm.row[tid] = own.x;
        sm.head[tid] = item.kv_head * a.group + m % a.group;
        sm.limit[tid] = !live ? 0 : item.start >= 0 ? own.y + 1 - item.start : item.keys;
    }
    compute_sync();
    const float *q = reinterpret_cast<const float *>(a.q);
    const bool aligned = !((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(a.ldq * 4)) & 15);
#pragma unroll 8
    for (int i = tid; i < rows * (HD / 4); i += kCompute) {
        const int r = i / (HD / 4), c = i % (HD / 4);
        float4 v = make_float4(0, 0, 0, 0);
        if (r < item.m && c * 4 < a.head_dim) {
            const float *from = q + (long long)sm.row[r] * a.ldq + sm.head[r] * a.head_dim + c * 4;
            v = aligned ? *reinterpret_cast<const float4 *>(from) : make_float4(from[0], from[1], from[2], from[3]);
        }
        const float f = a.scale_log2;
        *reinterpret_cast<float4 *>(&sm.q[q_chunk<HD, RI>(r, c)]) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    }
    compute_sync();
}

template <int HD, typename Wait>
__device__ void few_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item, Smem<HD> &sm, Ring<HD> &ring, Wait &wait)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    load_rows<HD, kTileM>(a, plan, item, sm, kFewRows);
    const bool works = lane * 4 < HD;                  // this lane's 4 columns exist
    const int chunk = works ? lane : 0, k0 = warp * 8;
    // After the exchange: this lane's key of the warp's 8, and its two rows.
    const int own_key = k0 + (lane >> 2), row0 = (lane & 3) * 2;
    const int limit0 = sm.limit[row0], limit1 = sm.limit[row0 + 1], least = sm.limit[0];
    float4 q[kFewRows];
    float2 acc[kFewRows][2];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        q[r] = works ? *reinterpret_cast<const float4 *>(&sm.q[q_chunk<HD, kTileM>(r, lane)]) : make_float4(0, 0, 0, 0);
        acc[r][0] = acc[r][1] = make_float2(0, 0);
    }
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0, l1 = 0;
    float (&w)[kFewRows + 1][kFewRows] = sm.few[warp];
    for (int j = 0; j < item.blocks; ++j) {
        const int t0 = (item.block0 + j) * kBlock;
        // ---- scores
        wait(&sm.full[ring.stage], ring.parity);
        const uint8_t *tile = sm.stages[ring.stage];
        float s[2];
        {
            const bool upper = lane & 16, mid = lane & 8, low = lane & 4, row_hi = lane & 2, row_lo = lane & 1;
            auto dots = [&](int key, float (&d)[kFewRows]) {
                const float4 k = tile_chunk(tile, k0 + key, chunk);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) {
                    const float2 t = __ffma2_rn(hi2(q[r]), hi2(k), __fmul2_rn(lo2(q[r]), lo2(k)));
                    d[r] = t.x + t.y;
                }
            };
            // The lanes with `mine` set keep b of (a, b), the others a, each summed with its partner's.
            auto meet = [&](bool mine, int mask, float a, float b) {
                return (mine ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, mine ? a : b, mask);
            };
            float quarter[2][kFewRows];
#pragma unroll
            for (int e = 0; e < 2; ++e) {              // key bit 0
                float half[2][kFewRows];
#pragma unroll
                for (int g = 0; g < 2; ++g) {          // key bit 1
                    float a[kFewRows], b[kFewRows];
                    dots(e + 2 * g, a);
                    dots(e + 2 * g + 4, b);
#pragma unroll
                    for (int r = 0; r < kFewRows; ++r) half[g][r] = meet(upper, 16, a[r], b[r]);
                }
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) quarter[e][r] = meet(mid, 8, half[0][r], half[1][r]);
            }
            float rows[kFewRows], four[4];
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) rows[r] = meet(low, 4, quarter[0][r], quarter[1][r]);
#pragma unroll
            for (int r = 0; r < 4; ++r) four[r] = meet(row_hi, 2, rows[r], rows[r + 4]);
#pragma unroll
            for (int r = 0; r < 2; ++r) s[r] = meet(row_lo, 1, four[r], four[r + 2]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
        // ---- weights
        const float s0 = t0 + own_key < limit0 ? s[0] : -INFINITY, s1 = t0 + own_key < limit1 ? s[1] : -INFINITY;
        float top0 = s0, top1 = s1;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, o));
            top1 = fmaxf(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, o));
        }
        top0 = fmaxf(top0, m0);
        top1 = fmaxf(top1, m1);
        const bool grown = top0 > m0 || top1 > m1;
        const float base0 = top0 == -INFINITY ? 0.0f : top0, base1 = top1 == -INFINITY ? 0.0f : top1;
        const float p0 = exp2f(s0 - base0), p1 = exp2f(s1 - base1);
        *reinterpret_cast<float2 *>(&w[lane >> 2][row0]) = make_float2(p0, p1);
        if (__any_sync(0xFFFFFFFFu, grown)) {
            const float keep0 = exp2f(m0 - base0), keep1 = exp2f(m1 - base1);
            l0 *= keep0;
            l1 *= keep1;
            if (lane < 4) *reinterpret_cast<float2 *>(&w[kFewRows][row0]) = make_float2(keep0, keep1);
            __syncwarp();
            const float4 fa = *reinterpret_cast<const float4 *>(&w[kFewRows][0]), fb = *reinterpret_cast<const float4 *>(&w[kFewRows][4]);
            const float f[kFewRows] = {fa.x, fa.y, fa.z, fa.w, fb.x, fb.y, fb.z, fb.w};
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                acc[r][0] = __fmul2_rn(acc[r][0], both(f[r]));
                acc[r][1] = __fmul2_rn(acc[r][1], both(f[r]));
            }
        }
        m0 = top0;
        m1 = top1;
        l0 += p0;                                      // this lane's keys only; the lanes are added at the end
        l1 += p1;
        __syncwarp();
        // ---- outputs
        wait(&sm.full[ring.stage], ring.parity);
        tile = sm.stages[ring.stage];
        // Rows that do not see a key skip it, whatever V holds there (the tile's rows behind the segment's keys
        // hold anything).
        const bool masked = t0 + k0 + 8 > least || t0 + k0 + 8 > item.keys;
        auto add = [&](int key, auto seen) {
            const float4 v = tile_chunk(tile, k0 + key, chunk);
            const float4 wa = *reinterpret_cast<const float4 *>(&w[key][0]), wb = *reinterpret_cast<const float4 *>(&w[key][4]);
            const float f[kFewRows] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                if (!seen(r)) continue;
                acc[r][0] = __ffma2_rn(both(f[r]), lo2(v), acc[r][0]);
                acc[r][1] = __ffma2_rn(both(f[r]), hi2(v), acc[r][1]);
            }
        };
        if (!masked) {
#pragma unroll
            for (int key = 0; key < 8; ++key) add(key, [](int) { return true; });
        } else {
#pragma unroll 1
            for (int key = 0; key < min(8, item.keys - t0 - k0); ++key)
                add(key, [&](int r) { return t0 + k0 + key < sm.limit[r]; });
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
    }
    // Merge the warps: their accumulators lie behind the 8 query rows.
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, o);
        l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, o);
    }
    float *merged = &sm.q[kFewRows * HD];              // [warp][row][HD]
    static_assert(kWarps * kFewRows <= kTileM - kFewRows, "room");
    if (lane < 4) {
        *reinterpret_cast<float2 *>(&sm.few_m[warp][row0]) = make_float2(m0, m1);
        *reinterpret_cast<float2 *>(&sm.few_l[warp][row0]) = make_float2(l0, l1);
    }
    if (works)
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
            *reinterpret_cast<float4 *>(&merged[(warp * kFewRows + r) * HD + lane * 4]) = make_float4(acc[r][0].x, acc[r][0].y, acc[r][1].x, acc[r][1].y);
    compute_sync();
    const int r = warp;                                // warp r merges row r
    if (r < item.m) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.few_m[w][r]);
        const float base = top == -INFINITY ? 0.0f : top;
        float weight[kWarps], sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            weight[w] = exp2f(sm.few_m[w][r] - base);
            sum = fmaf(sm.few_l[w][r], weight[w], sum);
        }
        for (int d = lane; d < a.head_dim; d += 32) {
            float o = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) o = fmaf(merged[(w * kFewRows + r) * HD + d], weight[w], o);
            if (item.direct)
                store_out(a, sm.row[r], sm.head[r], d, o / sum);
            else
                plan->part_o[((long long)item.slot * kTileM + r) * a.head_dim + d] = o;
        }
        if (!item.direct && lane == 0) plan->part_ml[(long long)item.slot * kTileM + r] = make_float2(top, sum);
    }
    compute_sync();
}

template <int HD, int RI, typename Wait>
__device__ void many_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item, Smem<HD> &sm, Ring<HD> &ring, Wait &wait)
{
    constexpr int OC = (HD + 63) / 64;                 // groups of 4 output columns per thread
    const int tid = threadIdx.x, lane = tid & 31, tx = tid & 15, ty = tid >> 4;
    load_rows<HD, RI>(a, plan, item, sm, RI * 16);
    float m[RI], l[RI];
    float2 acc[RI][OC][2];
    int limit[RI];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        limit[i] = sm.limit[ty * RI + i];
        m[i] = -INFINITY;
        l[i] = 0;
#pragma unroll
        for (int c = 0; c < OC; ++c) acc[i][c][0] = acc[i][c][1] = make_float2(0, 0);
    }
    const int least = sm.limit[0];
    for (int block = item.block0; block < item.block0 + item.blocks; ++block) {
        const int t0 = block * kBlock;
        wait(&sm.full[ring.stage], ring.parity);
        const uint8_t *tile = sm.stages[ring.stage];
        float2 s2[RI][4];
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0, 0);
#pragma unroll 4
        for (int c = 0; c < HD / 4; ++c) {
            float4 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = tile_chunk(tile, tx + 16 * j, c);
#pragma unroll
            for (int i = 0; i < RI; ++i) {
                const float4 q = *reinterpret_cast<const float4 *>(&sm.q[q_chunk<HD, RI>(ty * RI + i, c)]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s2[i][j] = __ffma2_rn(lo2(q), lo2(k[j]), s2[i][j]);
                    s2[i][j] = __ffma2_rn(hi2(q), hi2(k[j]), s2[i][j]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
#pragma unroll
        for (int i = 0; i < RI; ++i) {
            float s[4], top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = t0 + tx + 16 * j < limit[i] ? s2[i][j].x + s2[i][j].y : -INFINITY;
                top = fmaxf(top, s[j]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m[i] - base);
            m[i] = top;
            float sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[j] - base);
                sum += p;
                sm.p[p_at<RI>(ty * RI + i, tx + 16 * j)] = p;
            }
            l[i] = fmaf(l[i], keep, sum);              // this thread's keys only
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                acc[i][c][0] = __fmul2_rn(acc[i][c][0], both(keep));
                acc[i][c][1] = __fmul2_rn(acc[i][c][1], both(keep));
            }
        }
        __syncwarp();                                  // a warp's rows of weights are its own
        wait(&sm.full[ring.stage], ring.parity);
        tile = sm.stages[ring.stage];
        // Rows that do not see a key skip it, whatever V holds there (the tile's rows behind the segment's keys
        // hold anything).
        auto add = [&](int key, const float (&w)[RI], auto seen) {
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                if (HD % 64 && c * 16 + tx >= HD / 4) continue;
                const float4 v = tile_chunk(tile, key, c * 16 + tx);
#pragma unroll
                for (int i = 0; i < RI; ++i) {
                    if (!seen(i)) continue;
                    acc[i][c][0] = __ffma2_rn(both(w[i]), lo2(v), acc[i][c][0]);
                    acc[i][c][1] = __ffma2_rn(both(w[i]), hi2(v), acc[i][c][1]);
                }
            }
        };
        if (t0 + kBlock <= least && t0 + kBlock <= item.keys) {
#pragma unroll 2
            for (int t = 0; t < kBlock; t += 4) {
                float4 p[RI];
#pragma unroll
                for (int i = 0; i < RI; ++i) p[i] = *reinterpret_cast<const float4 *>(&sm.p[p_at<RI>(ty * RI + i, t)]);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float w[RI];
#pragma unroll
                    for (int i = 0; i < RI; ++i) w[i] = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                    add(t + u, w, [](int) { return true; });
                }
            }
        } else {
#pragma unroll 1
            for (int t = 0; t < min(kBlock, item.keys - t0); ++t) {
                float w[RI];
#pragma unroll
                for (int i = 0; i < RI; ++i) w[i] = sm.p[p_at<RI>(ty * RI + i, t)];
                add(t, w, [&](int i) { return t0 + t < limit[i]; });
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], o);
        const int r = ty * RI + i;
        if (r < item.m) {
            const float inverse = 1.0f / l[i];
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                if ((c * 16 + tx) * 4 >= a.head_dim) continue;
                const float v[4] = {acc[i][c][0].x, acc[i][c][0].y, acc[i][c][1].x, acc[i][c][1].y};
                const int d = (c * 16 + tx) * 4;
                if (item.direct) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) store_out(a, sm.row[r], sm.head[r], d + e, v[e] * inverse);
                } else {
                    *reinterpret_cast<float4 *>(&plan->part_o[((long long)item.slot * kTileM + r) * a.head_dim + d]) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
            if (!item.direct && tx == 0) plan->part_ml[(long long)item.slot * kTileM + r] = make_float2(m[i], l[i]);
        }
    }
    compute_sync();
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) f32_attention_kernel(const Args t, const __grid_constant__ CUtensorMap map)
{
    typedef Layout<HD> L;
    const BatchAttn &a = t.a;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<HD> &sm = *reinterpret_cast<Smem<HD> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5;
    if (smem_u32(smem_raw) & 1023u) {          // the swizzle needs it; dynamic shared memory starts there
        if (tid == 0) atomicOr(a.err, kDevErrTimeout);
        return;
    }
    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kWarps);
        }
        sm.abort = 0;
        fence_mbar_init();
        prefetch_tensormap(&map);
    }
    __syncthreads();
    pdl_wait();
    const DevPlan *plan = a.plan;
    const int first = plan_array<int>(plan, plan->cta_off)[blockIdx.x], last = plan_array<int>(plan, plan->cta_off)[blockIdx.x + 1];
    // An expired wait is recorded and ends all others at once; the compute warps, which meet at barriers, go on to
    // their end with whatever the tiles hold.
    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {
        if (mbar_test(b, parity)) return true;
        if (sm.abort) return false;
        if (mbar_wait_bounded(b, parity)) return true;
        atomicOr(a.err, kDevErrTimeout);
        sm.abort = 1;
        return false;
    };
    Ring<HD> ring;
    if (warp >= kWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoaderRegs));
        if (warp == kWarps && elect_one()) {
            int units = 0;
            bool ok = true;
            for (int i = first; i < last && ok; ++i) {
                const PlanItem item = load_item(plan, i);
                const int *pages = plan_array<int>(plan, plan->pages) + item.page_off;
                ok = a.page_tokens >= kBlock  ? load_tiles<HD, 1>(t, map, sm, pages, item, ring, units, wait)
                     : a.page_tokens == 32    ? load_tiles<HD, 2>(t, map, sm, pages, item, ring, units, wait)
                                              : load_tiles<HD, 4>(t, map, sm, pages, item, ring, units, wait);
            }
            // The copies in flight land before the CTA may end.
            if (!ok)
                for (int u = max(0, units - L::kStages); u < units; ++u)
                    mbar_wait_bounded(&sm.full[u % L::kStages], (uint32_t)((u / L::kStages) & 1));
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
        for (int i = first; i < last; ++i) {
            const PlanItem item = load_item(plan, i);
            if (item.m <= kFewRows)
                few_rows<HD>(a, plan, item, sm, ring, wait);
            else if (item.m <= 64)
                many_rows<HD, 4>(a, plan, item, sm, ring, wait);
            else if (item.m <= 96)
                many_rows<HD, 6>(a, plan, item, sm, ring, wait);
            else
                many_rows<HD, 8>(a, plan, item, sm, ring, wait);
        }
    }
    __syncthreads();
}

template <int HD>
cudaError_t launch(const Args &t, const CUtensorMap &map, cudaStream_t stream)
{
    static_assert(sizeof(Smem<HD>) <= 232448, "shared memory");
    cudaError_t e = opt_in_smem(reinterpret_cast<const void *>(&f32_attention_kernel<HD>), sizeof(Smem<HD>));
    if (e != cudaSuccess) return e;
    return launch_overlapped(f32_attention_kernel<HD>, dim3((unsigned)t.a.ctas), kThreads, sizeof(Smem<HD>), stream, t, map);
}

}  // namespace

bool f32_attention_takes(int type, int head_dim)
{
    return type == SATORI_F32 && head_dim <= 128;
}

void f32_plan_shape(int head_dim, int sm_count, PlanShape &shape)
{
    shape.tile_m = kTileM;
    shape.block = kBlock;
    shape.ctas = sm_count;
    shape.solo_m = kFewRows;
    // Hundreds of clocks: a block's bytes at an SM's share of HBM, its products on the FP32 units, an item's start
    // and end.
    shape.solo_cost = std::max(1, 30 * head_dim / 128);
    shape.pair_cost = std::max(1, 140 * head_dim / 128);
    shape.more_cost = 140 * head_dim / 128;
    shape.item_cost = 60;
    shape.slots_per_item = 1;
}

int f32_record_rows() { return kTileM; }

cudaError_t launch_f32_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream)
{
    const Args t = {a, layer_block};
    return a.head_dim <= 32   ? launch<32>(t, map, stream)
           : a.head_dim <= 64 ? launch<64>(t, map, stream)
           : a.head_dim <= 96 ? launch<96>(t, map, stream)
                              : launch<128>(t, map, stream);
}

}  // namespace satori
