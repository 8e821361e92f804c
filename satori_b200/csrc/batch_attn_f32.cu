// batch_attn_f32.cu -- attention of a batch over a paged FP32 cache with heads of 32, 64, 96 or 128, on the FP32
// units (the tensor cores would round its products).
//
// The formulas are the FP32-unit kernel's for other caches (one pass over the keys, running maximum and sum);
// here the keys come through a ring of shared memory tiles, so that the loads of the next blocks run under the
// arithmetic of this one.  One CTA per SM works through its share of the plan's items; warp 8's elected thread
// loads each block of 64 keys as a K and a V tile (TMA, 32 columns of 128 bytes a row with the 128-byte swizzle:
// 8 threads that read 16 bytes of 8 consecutive rows, or of one row, meet 8 different bank groups), warps 0-7
// compute:
//  * tiles of at most 8 rows (the query heads of one KV head of one request): for the scores a lane owns a key
//    and its warp two rows, so that a dot product needs no exchange; for the outputs a warp owns 8 keys, with a
//    running maximum of its own.  HBM bounds it (64 KB a block of 128-wide heads against about 1000 issue slots).
//  * tiles of up to 64 rows (a shared prefix, a prompt): 4 x 4 scores and 4 x HD / 16 outputs per thread.  The
//    FP32 units bound it: 8192 clocks a block at 128 columns.
// Products are packed two to an instruction (FFMA2), which halves the issue slots, not the arithmetic.
//
// Measured, 32 heads of 128 over 8 KV heads, against the kernel for other caches on the same call: one request of
// 300 tokens 11.1 us (20 us there, where each warp waits for its own loads), 16 requests that share 8192 tokens
// 51 us (55 us there), of which the FP32 units are busy about 30 us.
#include "batch.cuh"
#include "common.cuh"

#include <algorithm>

namespace satori {

namespace {

constexpr int kWarps = 8, kCompute = kWarps * 32, kThreads = kCompute + 32;
constexpr int kTileM = 64, kBlock = 64, kFewRows = 8;

template <int HD>
struct Layout {
    static constexpr int kSub = kBlock * 128;                      // 64 rows of 32 columns
    static constexpr int kTile = kSub * (HD / 32);
    static constexpr int kStages = HD <= 64 ? 8 : HD <= 96 ? 6 : 5;
};

template <int HD>
struct alignas(1024) Smem {
    uint8_t stages[Layout<HD>::kStages][Layout<HD>::kTile];
    float q[kTileM][HD + 4];
    union {
        float p[kTileM][kBlock + 4];
        struct {
            float s[2][kBlock][kFewRows];              // scores of a block, two buffers
            float w[kWarps][kFewRows + 1][kFewRows];   // a warp's weights [key][row], then the rows' factors
        } few;
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
            if (PER == 1) {
                load_4d(to, &map, key0 & mask, block0 + id[0] * page_blocks, full);
            } else {
#pragma unroll
                for (int b = 0; b < PER; ++b)
                    if (b < boxes)
#pragma unroll
                        for (int c = 0; c < HD / 32; ++c)
                            load_3d(to + c * L::kSub + b * kBox * 128, &map, c * 32, 0, block0 + id[b] * page_blocks, full);
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
template <int HD>
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
    for (int i = tid; i < rows * HD; i += kCompute) {
        const int r = i / HD, d = i % HD;
        sm.q[r][d] = r < item.m ? reinterpret_cast<const float *>(a.q)[(long long)sm.row[r] * a.ldq + sm.head[r] * HD + d] * a.scale_log2 : 0.0f;
    }
    compute_sync();
}

template <int HD, typename Wait>
__device__ void few_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item, Smem<HD> &sm, Ring<HD> &ring, Wait &wait)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    load_rows<HD>(a, plan, item, sm, kFewRows);
    const int half = warp & 1, r0 = warp & ~1;         // scores: this warp's 32 keys and rows r0, r0 + 1
    const bool scores = r0 < item.m;
    const int row8 = lane & 7, least = sm.limit[0];
    const int own_limit = sm.limit[row8];
    const bool works = lane * 4 < HD;
    float m = -INFINITY, l = 0;                        // row row8 over this warp's keys (four lanes alike)
    float2 acc[kFewRows][2];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) acc[r][0] = acc[r][1] = make_float2(0, 0);
    for (int j = 0; j < item.blocks; ++j) {
        const int t0 = (item.block0 + j) * kBlock, buffer = j & 1;
        // ---- scores
        wait(&sm.full[ring.stage], ring.parity);
        if (scores) {
            const int key = half * 32 + lane;
            const uint8_t *tile = sm.stages[ring.stage];
            float2 s0 = make_float2(0, 0), s1 = s0, u0 = s0, u1 = s0;
#pragma unroll 8
            for (int c = 0; c < HD / 4; ++c) {
                const float4 k = tile_chunk(tile, key, c);
                const float4 qa = *reinterpret_cast<const float4 *>(&sm.q[r0][c * 4]);
                const float4 qb = *reinterpret_cast<const float4 *>(&sm.q[r0 + 1][c * 4]);
                s0 = __ffma2_rn(lo2(qa), lo2(k), s0);
                u0 = __ffma2_rn(hi2(qa), hi2(k), u0);
                s1 = __ffma2_rn(lo2(qb), lo2(k), s1);
                u1 = __ffma2_rn(hi2(qb), hi2(k), u1);
            }
            const float2 a0 = __fadd2_rn(s0, u0), a1 = __fadd2_rn(s1, u1);
            *reinterpret_cast<float2 *>(&sm.few.s[buffer][key][r0]) = make_float2(a0.x + a0.y, a1.x + a1.y);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
        compute_sync();
        // ---- weights of this warp's 8 keys: lane (key & 3, row)
        const int k0 = warp * 8, ka = k0 + (lane >> 3);
        float sa = row8 < item.m && t0 + ka < own_limit ? sm.few.s[buffer][ka][row8] : -INFINITY;
        float sb = row8 < item.m && t0 + ka + 4 < own_limit ? sm.few.s[buffer][ka + 4][row8] : -INFINITY;
        float top = fmaxf(sa, sb);
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
        top = fmaxf(top, m);
        const float base = top == -INFINITY ? 0.0f : top;
        const float keep = exp2f(m - base), pa = exp2f(sa - base), pb = exp2f(sb - base);
        m = top;
        l = fmaf(l, keep, pa + pb);                    // this lane's keys only; the four lanes are added at the end
        sm.few.w[warp][lane >> 3][row8] = pa;
        sm.few.w[warp][(lane >> 3) + 4][row8] = pb;
        if (lane < 8) sm.few.w[warp][8][lane] = keep;
        __syncwarp();
        {
            const float4 ka4 = *reinterpret_cast<const float4 *>(&sm.few.w[warp][8][0]);
            const float4 kb4 = *reinterpret_cast<const float4 *>(&sm.few.w[warp][8][4]);
            const float f[8] = {ka4.x, ka4.y, ka4.z, ka4.w, kb4.x, kb4.y, kb4.z, kb4.w};
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                acc[r][0] = __fmul2_rn(acc[r][0], both(f[r]));
                acc[r][1] = __fmul2_rn(acc[r][1], both(f[r]));
            }
        }
        // ---- outputs: lane owns 4 columns
        wait(&sm.full[ring.stage], ring.parity);
        const uint8_t *tile = sm.stages[ring.stage];
        const bool masked = t0 + k0 + 8 > least;       // some row does not see some of these keys
        const int have = item.keys - t0;               // (the tile's rows from there on hold anything)
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            if (k0 + kk >= have) break;
            const float4 v = works ? tile_chunk(tile, k0 + kk, lane) : make_float4(0, 0, 0, 0);
            const float4 wa = *reinterpret_cast<const float4 *>(&sm.few.w[warp][kk][0]);
            const float4 wb = *reinterpret_cast<const float4 *>(&sm.few.w[warp][kk][4]);
            const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                if (masked && t0 + k0 + kk >= sm.limit[r]) continue;           // whatever V holds there
                acc[r][0] = __ffma2_rn(both(w[r]), lo2(v), acc[r][0]);
                acc[r][1] = __ffma2_rn(both(w[r]), hi2(v), acc[r][1]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
    }
    // Merge the warps: their accumulators lie behind the 8 query rows, over the scores.
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
    compute_sync();
    float *merged = &sm.q[kFewRows][0];                // [warp][row][HD]
    static_assert(sizeof(float) * kWarps * kFewRows * HD <= sizeof(float) * (kTileM - kFewRows) * (HD + 4) + sizeof(float) * kTileM * (kBlock + 4), "room");
    if (lane < 8) {
        sm.few_m[warp][lane] = m;
        sm.few_l[warp][lane] = l;
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
        for (int d = lane; d < HD; d += 32) {
            float o = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) o = fmaf(merged[(w * kFewRows + r) * HD + d], weight[w], o);
            if (item.direct)
                store_out(a, sm.row[r], sm.head[r], d, o / sum);
            else
                plan->part_o[((long long)item.slot * kTileM + r) * HD + d] = o;
        }
        if (!item.direct && lane == 0) plan->part_ml[(long long)item.slot * kTileM + r] = make_float2(top, sum);
    }
    compute_sync();
}

template <int HD, typename Wait>
__device__ void many_rows(const BatchAttn &a, const DevPlan *plan, const PlanItem &item, Smem<HD> &sm, Ring<HD> &ring, Wait &wait)
{
    constexpr int OC = (HD + 63) / 64;                 // groups of 4 output columns per thread
    const int tid = threadIdx.x, lane = tid & 31, tx = tid & 15, ty = tid >> 4;
    load_rows<HD>(a, plan, item, sm, kTileM);
    float m[4], l[4];
    float2 acc[4][OC][2];
    int limit[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        limit[i] = sm.limit[ty * 4 + i];
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
        float2 s2[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0, 0);
#pragma unroll 4
        for (int c = 0; c < HD / 4; ++c) {
            float4 q[4], k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4 *>(&sm.q[ty * 4 + i][c * 4]);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = tile_chunk(tile, tx + 16 * j, c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s2[i][j] = __ffma2_rn(lo2(q[i]), lo2(k[j]), s2[i][j]);
                    s2[i][j] = __ffma2_rn(hi2(q[i]), hi2(k[j]), s2[i][j]);
                }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
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
                sm.p[ty * 4 + i][tx + 16 * j] = p;
            }
            l[i] = fmaf(l[i], keep, sum);              // this thread's keys only
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                acc[i][c][0] = __fmul2_rn(acc[i][c][0], both(keep));
                acc[i][c][1] = __fmul2_rn(acc[i][c][1], both(keep));
            }
        }
        __syncwarp();                                  // a warp's 8 rows of weights are its own
        wait(&sm.full[ring.stage], ring.parity);
        tile = sm.stages[ring.stage];
        const bool masked = t0 + kBlock > least;       // some row does not see some key of the block
        const int have = min(kBlock, item.keys - t0);  // (the tile's rows from there on hold anything)
#pragma unroll 2
        for (int t = 0; t < have; t += 4) {
            float4 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4 *>(&sm.p[ty * 4 + i][t]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (t + u >= have) break;
#pragma unroll
                for (int c = 0; c < OC; ++c) {
                    if (HD % 64 && c * 16 + tx >= HD / 4) continue;
                    const float4 v = tile_chunk(tile, t + u, c * 16 + tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                        if (masked && t0 + t + u >= limit[i]) continue;        // whatever V holds there
                        acc[i][c][0] = __ffma2_rn(both(w), lo2(v), acc[i][c][0]);
                        acc[i][c][1] = __ffma2_rn(both(w), hi2(v), acc[i][c][1]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[ring.stage]);
        ring.next();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], o);
        const int r = ty * 4 + i;
        if (r < item.m) {
            const float inverse = 1.0f / l[i];
#pragma unroll
            for (int c = 0; c < OC; ++c) {
                if (HD % 64 && c * 16 + tx >= HD / 4) continue;
                const float v[4] = {acc[i][c][0].x, acc[i][c][0].y, acc[i][c][1].x, acc[i][c][1].y};
                const int d = (c * 16 + tx) * 4;
                if (item.direct) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) store_out(a, sm.row[r], sm.head[r], d + e, v[e] * inverse);
                } else {
                    *reinterpret_cast<float4 *>(&plan->part_o[((long long)item.slot * kTileM + r) * HD + d]) = make_float4(v[0], v[1], v[2], v[3]);
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
    if (warp == kWarps) {
        if (elect_one()) {
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
        for (int i = first; i < last; ++i) {
            const PlanItem item = load_item(plan, i);
            if (item.m <= kFewRows)
                few_rows<HD>(a, plan, item, sm, ring, wait);
            else
                many_rows<HD>(a, plan, item, sm, ring, wait);
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
    return type == SATORI_F32 && head_dim % 32 == 0 && head_dim <= 128;
}

void f32_plan_shape(int head_dim, int sm_count, PlanShape &shape)
{
    shape.tile_m = kTileM;
    shape.block = kBlock;
    shape.ctas = sm_count;
    shape.solo_m = kFewRows;
    // Hundreds of clocks: a block's bytes at HBM's share, its products on the FP32 units, an item's start and end.
    shape.solo_cost = std::max(1, 28 * head_dim / 128);
    shape.pair_cost = std::max(1, 100 * head_dim / 128);
    shape.item_cost = 60;
    shape.slots_per_item = 1;
}

int f32_record_rows() { return kTileM; }

cudaError_t launch_f32_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream)
{
    const Args t = {a, layer_block};
    switch (a.head_dim) {
    case 32: return launch<32>(t, map, stream);
    case 64: return launch<64>(t, map, stream);
    case 96: return launch<96>(t, map, stream);
    default: return launch<128>(t, map, stream);
    }
}

}  // namespace satori
