// batch_attn_tensor.cu -- attention of a batch over a paged 16-bit cache on the 5th-generation tensor cores
// (heads of 64 and 128).
//
// The same one pass over the keys as the FP32-unit kernel, as two matrix products per block of 64 keys:
// S = Q K^T and O += P V with P = 2^(s - m).  One CTA per SM works through its share of the plan's items:
//  * warp 8 loads the pages of a block's K and V with TMA (one box per page and 64 columns, 128-byte swizzle)
//    into a ring of stages;
//  * one lane of warp 9 issues the MMAs: S from shared memory (Q and K, both K-major), O with P from tensor
//    memory and V from shared memory as it lies (MN-major);
//  * warp 10 clears the rows of V behind a tile's last key;
//  * warps 0-3 and 4-7 are two softmax groups, each with its own O and two S / P buffers in tensor memory; a
//    thread owns one row.  A large tile (129..256 rows) gives each group 128 of its rows and every K and V
//    block serves both; a small one gives each group every other block.  The scores of a group's next block
//    are computed while it takes the exponentials of this one.
// The maximum that the exponentials refer to is raised only when it is exceeded by more than 2^8, so the
// accumulator in tensor memory is rescaled a few times per row, not at every block; P stays below 2^8 and the
// result does not depend on it.  P is rounded to the cache's type (half a step, as the operands already are);
// S, the sums and O are FP32.
//
// What bounds it: HBM for up to about 256 rows per block of keys, beyond that the exponentials (16 per clock
// and SM, 2048 clocks for two tiles' block) and the MMAs (2048 clocks) about equally.
#include "batch.cuh"
#include "common.cuh"

#include <algorithm>

namespace satori {

namespace {

constexpr int kTileRows = 128, kBlockKeys = 64;
constexpr int kSoftmaxThreads = 256, kThreads = kSoftmaxThreads + 96;
constexpr float kLazy = 8.0f;                  // log2 of what a weight may exceed 1 by

template <int HD>
struct Layout {
    static constexpr int kQHalf = kTileRows * 128, kHalf = kBlockKeys * 128;       // rows of 64 columns
    static constexpr int kQTile = kQHalf * (HD / 64), kTile = kHalf * (HD / 64);   // Q; K or V
    static constexpr int kStages = HD == 128 ? 10 : 20;
    static constexpr int kHeader = 1024;
    static constexpr int kBytes = kHeader + 2 * kQTile + kStages * kTile + 1024;
    static constexpr int kOCol = 4 * kBlockKeys;                   // tensor memory: S / P buffers, then O
};

constexpr int kMaxStages = 20;
struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t s_full[2][2], p_ready[2][2], pv_done[2][2];           // [group][buffer]: blocks in turn
    uint64_t q_ready[2], tail_full, tail_clear, drained;
    uint32_t tmem;
    volatile int abort;
};
static_assert(sizeof(Barriers) <= 1024, "header");

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// True in one lane of the (converged) warp.  The compiler knows that a single thread is in the branch, and keeps
// the operands of the MMAs there in uniform registers; behind a comparison of the lane number it moves all of
// them there for every MMA (about 90 clocks each, more than the MMA takes).
__device__ __forceinline__ bool elect_one()
{
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b32 r;\n\telect.sync r|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(smem_u32(bar)) : "memory");
}

// Shared-memory matrix descriptors with the 128-byte swizzle (start, leading and stride byte offsets in 16-byte
// units, version 1, layout 2; the stride between groups of 8 rows is 1024): the high word is the same for all,
// and a start `b` bytes further is b / 16 more in the low word.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
__device__ __forceinline__ uint64_t desc(uint32_t low) { return (uint64_t)kDescHigh << 32 | low; }

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(desc(a)), "l"(desc(b)), "r"(idesc), "r"(add ? 1u : 0u) : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(desc(b)), "r"(idesc), "r"(add ? 1u : 0u) : "memory");
}

__device__ __forceinline__ void tma_load_3d(void *dst, const void *map, int c0, int c1, int c2, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
                 : "memory");
}

#define SATORI_R8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), \
                        "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define SATORI_W8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), \
                        "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])

// 32 columns of the warp's 32 tensor memory lanes; the caller waits.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : SATORI_R8(v, 0), SATORI_R8(v, 8), SATORI_R8(v, 16), SATORI_R8(v, 24)
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::SATORI_W8(v, 0), SATORI_W8(v, 8), SATORI_W8(v, 16), SATORI_W8(v, 24), "r"(addr) : "memory");
}
// The loaded registers pass through the wait, so that nothing reads them before it.
#define SATORI_U8(v, i) "+r"((v)[i]), "+r"((v)[i + 1]), "+r"((v)[i + 2]), "+r"((v)[i + 3]), "+r"((v)[i + 4]), \
                        "+r"((v)[i + 5]), "+r"((v)[i + 6]), "+r"((v)[i + 7])
__device__ __forceinline__ void tmem_wait_load(uint32_t *v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : SATORI_U8(v, 0), SATORI_U8(v, 8), SATORI_U8(v, 16), SATORI_U8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float x, float y)
{
    if (TYPE == SATORI_F16) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&b);
}

// Scores of keys `see` and above of 32 are not the row's to see.
__device__ __forceinline__ void mask_scores(uint32_t *s, int see)
{
    if (see < 32) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (e >= see) s[e] = 0xFF800000u;
    }
    __syncwarp();
}

struct TensorArgs {
    BatchAttn a;
    int layer_block;                 // first (page, K or V, head) block of the layer
    int wide_q, wide_out;            // 16-byte accesses of q and out rows are possible
};

// A role's view of one item.
struct Work {
    PlanItem item;
    bool pair;
    // Blocks of each softmax group, and how many blocks ahead of O the scores run.  An item's loads are in the
    // order of use: the leading blocks' K, then V and the next K in turn.
    __device__ __forceinline__ int blocks(int g) const { return pair ? item.blocks : (item.blocks + 1 - g) / 2; }
    __device__ __forceinline__ int lead() const { return min(item.blocks, pair ? 2 : 4); }
    // Keys of the item's last block, when the tile ends inside it; 0: no row of V needs clearing.
    __device__ __forceinline__ int tail() const
    {
        const int have = item.keys - (item.block0 + item.blocks - 1) * kBlockKeys;
        return have < kBlockKeys ? have : 0;
    }
};

// A place in the ring of stages, and the parity of its turn.
template <int NS>
struct Ring {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next()
    {
        if (++stage == NS) {
            stage = 0;
            parity ^= 1u;
        }
    }
    __device__ __forceinline__ void advance(int n)
    {
        const int to = stage + n;
        parity ^= (uint32_t)(to / NS) & 1u;
        stage = to % NS;
    }
};

__device__ __forceinline__ Work load_work(const DevPlan *plan, int i)
{
    Work w;
    const int4 *src = reinterpret_cast<const int4 *>(plan_array<PlanItem>(plan, plan->items) + i);
    int4 *dst = reinterpret_cast<int4 *>(&w.item);
#pragma unroll
    for (int k = 0; k < (int)(sizeof(PlanItem) / 16); ++k) dst[k] = __ldg(src + k);
    w.pair = w.item.m > kTileRows;
    return w;
}

// 32 columns of a row's accumulator: its share of the partial record, or of the output.
template <int TYPE, int HD>
__device__ __forceinline__ void store_output(const TensorArgs &t, const DevPlan *plan, const Work &w, uint32_t *o,
                                             float inverse, int row, int head, long long record, int c)
{
    typedef typename Elem<TYPE>::type T;
    const BatchAttn &a = t.a;
    if (!w.item.direct) {
        // [column / 4][row]: the warp's rows are neighbours.
        const int r = (int)(record % kTileRows);
        uint4 *dst = reinterpret_cast<uint4 *>(plan->part_o) + (record - r) * (HD / 4) + (c / 4) * kTileRows + r;
#pragma unroll
        for (int e = 0; e < 32; e += 4) dst[e / 4 * kTileRows] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        return;
    }
    const long long to = (long long)row * a.ldo + (long long)head * HD + c;
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inverse);
    if (a.out_f32) {
        float *dst = reinterpret_cast<float *>(a.out) + to;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            if (t.wide_out) {
                *reinterpret_cast<uint4 *>(dst + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
#pragma unroll
                for (int f = 0; f < 4; ++f) dst[e + f] = __uint_as_float(o[e + f]);
            }
        }
    } else {
        T *dst = reinterpret_cast<T *>(a.out) + to;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
            if (t.wide_out) {
                uint4 v;
                v.x = pack2<TYPE>(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                v.y = pack2<TYPE>(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                v.z = pack2<TYPE>(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]));
                v.w = pack2<TYPE>(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
                *reinterpret_cast<uint4 *>(dst + e) = v;
            } else {
#pragma unroll
                for (int f = 0; f < 8; ++f) dst[e + f] = Elem<TYPE>::from_float(__uint_as_float(o[e + f]));
            }
        }
    }
}

template <int TYPE, int HD>
__global__ void __launch_bounds__(kThreads, 1) tensor_attention_kernel(const TensorArgs t, const __grid_constant__ CUtensorMap map)
{
    typedef Layout<HD> L;
    typedef typename Elem<TYPE>::type T;
    constexpr int NS = L::kStages;
    const BatchAttn &a = t.a;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Barriers *bar = reinterpret_cast<Barriers *>(smem);
    uint8_t *q_tiles = smem + L::kHeader, *stages = q_tiles + 2 * L::kQTile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar->full[s], 1);
            mbar_init(&bar->empty[s], 1);
        }
        for (int g = 0; g < 2; ++g) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bar->s_full[g][b], 1);
                mbar_init(&bar->p_ready[g][b], kTileRows);
                mbar_init(&bar->pv_done[g][b], 1);
            }
            mbar_init(&bar->q_ready[g], kTileRows);
        }
        mbar_init(&bar->tail_full, 1);
        mbar_init(&bar->tail_clear, 32);
        mbar_init(&bar->drained, 1);
        bar->abort = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar->tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == 8 && lane == 0) prefetch_tensormap(&map);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bar->tmem;
    // Everything before came from the launch alone; the plan, q and the pages are other kernels' results.
    pdl_wait();
    const DevPlan *plan = a.plan;
    const int first = plan_array<int>(plan, plan->cta_off)[blockIdx.x];
    const int last = plan_array<int>(plan, plan->cta_off)[blockIdx.x + 1];
    // A wait that expires is recorded, and every role leaves at its next wait.
    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {
        if (mbar_test(b, parity)) return true;
        if (bar->abort) return false;
        if (mbar_wait_bounded(b, parity)) return true;
        atomicOr(a.err, kDevErrTimeout);
        bar->abort = 1;
        return false;
    };

    if (warp == 8) {
        // ---- loads
        const int box = min(a.page_tokens, kBlockKeys), shift = __ffs(a.page_tokens) - 1;
        // Lane l loads 64-column half l % (HD / 64) of box l / (HD / 64) of a block.
        const int b = lane / (HD / 64), half = lane % (HD / 64);
        Ring<NS> ring;
        int units = 0;
        bool ok = true;
        for (int i = first; i < last && ok; ++i) {
            const Work w = load_work(plan, i);
            const int *pages = plan_array<int>(plan, plan->pages) + w.item.page_off;
            auto load = [&](int j, int kv) {
                const int t0 = (w.item.block0 + j) * kBlockKeys, have = min(kBlockKeys, w.item.keys - t0);
                const int boxes = (have + box - 1) / box, key = t0 + b * box, s = ring.stage;
                const bool mine = b < boxes;
                const int page = mine ? __ldg(pages + (key >> shift)) : 0;
                ok = __all_sync(0xFFFFFFFFu, wait(&bar->empty[s], ring.parity ^ 1u));
                if (!ok) return;
                if (lane == 0) mbar_expect_tx(&bar->full[s], (uint32_t)(boxes * box * HD * 2));
                __syncwarp();
                if (mine)
                    tma_load_3d(stages + (size_t)s * L::kTile + half * L::kHalf + b * box * 128, &map, half * 64,
                                key & (a.page_tokens - 1), t.layer_block + (page * 2 + kv) * a.kv_heads + w.item.kv_head,
                                &bar->full[s]);
                ring.next();
                ++units;
            };
            const int lead = w.lead();
            for (int j = 0; j < lead && ok; ++j) load(j, 0);
            for (int j = 0; j < w.item.blocks && ok; ++j) {
                load(j, 1);
                if (ok && j + lead < w.item.blocks) load(j + lead, 0);
            }
        }
        if (!ok)      // the copies in flight land before the CTA may end
            for (int u = max(0, units - NS); u < units; ++u) mbar_wait_bounded(&bar->full[u % NS], (uint32_t)((u / NS) & 1));
    } else if (warp == 10) {
        // ---- V behind the last key: whatever the stage or the page holds there meets weights of zero, so it
        // must be finite.
        Ring<NS> ring;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = first; i < last && ok; ++i) {
            const Work w = load_work(plan, i);
            const int have = w.tail();
            ring.advance(2 * w.item.blocks - 1);       // the item's last load
            if (have > 0) {
                // Warp 9 has seen the load arrive, and waits: the stage keeps its contents meanwhile.
                ok = __all_sync(0xFFFFFFFFu, wait(&bar->tail_full, phase));
                if (!ok) break;
                phase ^= 1u;
                uint8_t *v = stages + (size_t)ring.stage * L::kTile + have * 128;
                for (int c = lane; c < (kBlockKeys - have) * 8; c += 32)
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h)
                        *reinterpret_cast<uint4 *>(v + h * L::kHalf + c * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&bar->tail_clear);
            }
            ring.next();
        }
    } else if (warp == 9) {
        // ---- matrix products
        if (elect_one()) {
            constexpr uint32_t kFormat = TYPE == SATORI_BF16 ? 1u : 0u;
            // FP32 accumulator, A and B of the cache's type, M = 128; S: N = 64, both K-major; O: N = HD, B MN-major.
            constexpr uint32_t kBase = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(kTileRows >> 4) << 24);
            constexpr uint32_t kDescS = kBase | ((uint32_t)(kBlockKeys >> 3) << 17);
            constexpr uint32_t kDescO = kBase | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
            const uint32_t q_low = desc_low(smem_u32(q_tiles), 16), k_low = desc_low(smem_u32(stages), 16);
            const uint32_t v_low = desc_low(smem_u32(stages), L::kHalf);
            Ring<NS> ring;
            uint32_t q_phase = 0, tail_phase = 0;      // bit g of q_phase: group g's parity
            int done0 = 0, done1 = 0;                  // blocks of each group so far
            bool ok = true, issued = false;
            for (int i = first; i < last && ok; ++i) {
                const Work w = load_work(plan, i);
                const int n = w.item.blocks, lead = w.lead();
                // S = Q K^T of the group's block number `at`.
                auto scores = [&](int g, int at, int stage) {
                    const uint32_t d = tmem + (g * 2 + (at & 1)) * kBlockKeys;
                    const uint32_t q = q_low + g * (L::kQTile >> 4), k = k_low + stage * (L::kTile >> 4);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma_ss(d, q + (ks / 4) * (L::kQHalf >> 4) + (ks % 4) * 2, k + (ks / 4) * (L::kHalf >> 4) + (ks % 4) * 2,
                               kDescS, ks > 0);
                    commit(&bar->s_full[g][at & 1]);
                };
                // O += P V, once P is there.
                auto values = [&](int g, int at, int stage, bool add) -> bool {
                    if (!wait(&bar->p_ready[g][at & 1], (uint32_t)(at >> 1) & 1u)) return false;
                    fence_after();
                    const uint32_t p = tmem + (g * 2 + (at & 1)) * kBlockKeys, v = v_low + stage * (L::kTile >> 4);
#pragma unroll
                    for (int ks = 0; ks < kBlockKeys / 16; ++ks)
                        mma_ts(tmem + L::kOCol + g * HD, p + ks * 8, v + ks * (2048 >> 4), kDescO, ks > 0 || add);
                    commit(&bar->pv_done[g][at & 1]);
                    return true;
                };
                // A small tile's group g has the blocks j = g, g + 2, ..; a large tile's groups have all of them.
                auto block_scores = [&](int j) -> bool {
                    if (!wait(&bar->full[ring.stage], ring.parity)) return false;
                    fence_after();
                    if (w.pair || (j & 1) == 0) scores(0, done0 + (w.pair ? j : j >> 1), ring.stage);
                    if (w.pair || (j & 1) == 1) scores(1, done1 + (w.pair ? j : j >> 1), ring.stage);
                    commit(&bar->empty[ring.stage]);
                    ring.next();
                    return true;
                };
                for (int g = 0; g < 2 && ok; ++g)
                    if (w.blocks(g) > 0) {
                        ok = wait(&bar->q_ready[g], q_phase >> g & 1);
                        q_phase ^= 1u << g;
                    }
                fence_after();
                issued = issued || ok;
                for (int j = 0; j < lead && ok; ++j) ok = block_scores(j);
                for (int j = 0; j < n && ok; ++j) {
                    const int sv = ring.stage, next = j + lead;
                    ok = wait(&bar->full[sv], ring.parity);
                    if (ok && j + 1 == n && w.tail() > 0) {
                        mbar_arrive(&bar->tail_full);
                        ok = wait(&bar->tail_clear, tail_phase);
                        tail_phase ^= 1u;
                    }
                    if (!ok) break;
                    ring.next();
                    if (w.pair) {
                        // Each group's next scores follow its own O at once, so that it does not wait for the other.
                        const int sk = ring.stage;
                        ok = values(0, done0 + j, sv, j > 0);
                        if (ok && next < n) {
                            ok = wait(&bar->full[sk], ring.parity);
                            if (!ok) break;
                            ring.next();
                            fence_after();
                            scores(0, done0 + next, sk);
                        }
                        ok = ok && values(1, done1 + j, sv, j > 0);
                        if (!ok) break;
                        commit(&bar->empty[sv]);
                        if (next < n) {
                            scores(1, done1 + next, sk);
                            commit(&bar->empty[sk]);
                        }
                    } else {
                        ok = (j & 1) ? values(1, done1 + (j >> 1), sv, j > 1) : values(0, done0 + (j >> 1), sv, j > 1);
                        if (!ok) break;
                        commit(&bar->empty[sv]);
                        if (next < n) ok = block_scores(next);
                    }
                }
                done0 += w.blocks(0);
                done1 += w.blocks(1);
            }
            // The issued MMAs finish before the tensor memory is freed.
            if (issued) {
                commit(&bar->drained);
                mbar_wait_bounded(&bar->drained, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: thread r of group g owns tile row r (and tensor memory lane r)
        const int g = warp >> 2, r = tid & (kTileRows - 1), quad = warp & 3;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t o_addr = lanes + L::kOCol + g * HD;
        uint8_t *q_tile = q_tiles + g * L::kQTile;
        int done = 0;                          // this group's blocks so far
        bool ok = true;
        for (int i = first; i < last && ok; ++i) {
            const Work w = load_work(plan, i);
            const int blocks = w.blocks(g);
            const int m = (w.pair ? g * kTileRows : 0) + r;
            const bool live = m < w.item.m;
            const long long record = (long long)(w.item.slot + g) * kTileRows + r;
            if (blocks == 0) {                 // a small tile's only block is the other group's
                if (live && !w.item.direct) plan->part_ml[record] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            int2 own = make_int2(0, 0);        // the row's number and position
            if (live)
                own = __ldg(reinterpret_cast<const int2 *>(plan_array<PlanRow>(plan, plan->seg_rows) + w.item.row_off) +
                            (w.item.m0 + m) / a.group);
            const int row = own.x, head = w.item.kv_head * a.group + (w.item.m0 + m) % a.group;
            const int limit = !live ? 0 : w.item.start >= 0 ? own.y + 1 - w.item.start : w.item.keys;
            // Q rows of this warp into shared memory, K-major with the 128-byte swizzle: 16-byte chunk c of row r
            // lies at chunk c ^ (r % 8).  All loads are in flight before the first store.
            {
                constexpr int PER_ROW = HD / 8, ROWS = 32 / PER_ROW, STEPS = 32 / ROWS;
                const long long q_off = live ? (long long)row * a.ldq + (long long)head * HD : -1;
                const int c = lane % PER_ROW;
                uint4 v[STEPS];
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const long long off = __shfl_sync(0xFFFFFFFFu, q_off, k * ROWS + lane / PER_ROW);
                    v[k] = make_uint4(0, 0, 0, 0);
                    const T *src = reinterpret_cast<const T *>(a.q) + off + c * 8;
                    if (off >= 0 && t.wide_q) {
                        v[k] = __ldg(reinterpret_cast<const uint4 *>(src));
                    } else if (off >= 0) {
                        const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
                        v[k] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16,
                                          h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
                    }
                }
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const int rr = quad * 32 + k * ROWS + lane / PER_ROW;
                    *reinterpret_cast<uint4 *>(q_tile + (c / 8) * L::kQHalf + rr * 128 + (((c & 7) ^ (rr & 7)) * 16)) = v[k];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&bar->q_ready[g]);

            const bool idle = __ballot_sync(0xFFFFFFFFu, live) == 0;       // the whole warp: rows behind the tile
            float ref = -INFINITY, sum = 0;    // ref: the maximum (log2 units) that the weights refer to
            for (int k = 0; k < blocks; ++k) {
                const int block = w.item.block0 + (w.pair ? k : 2 * k + g), at = done + k;
                const uint32_t s_addr = lanes + (g * 2 + (at & 1)) * kBlockKeys;
                ok = __all_sync(0xFFFFFFFFu, wait(&bar->s_full[g][at & 1], (uint32_t)(at >> 1) & 1u));
                if (!ok) break;
                fence_after();
                if (!idle) {
                    const int see = limit - block * kBlockKeys;            // keys of the block that the row sees
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    uint32_t s[2][32];
                    tmem_load32(s_addr, s[0]);
                    tmem_load32(s_addr + 32, s[1]);
                    tmem_wait_load(s[0]);
                    tmem_wait_load(s[1]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        mask_scores(s[c], see - c * 32);
#pragma unroll
                        for (int e = 0; e < 32; ++e) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(s[c][e]));
                    }
                    const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
                    const bool raise = high > ref + kLazy || (k == 0 && high > -INFINITY);
                    if (k > 0 && __any_sync(0xFFFFFFFFu, raise)) {
                        // The last block's product may still be adding to O.
                        ok = __all_sync(0xFFFFFFFFu, wait(&bar->pv_done[g][(at - 1) & 1], (uint32_t)((at - 1) >> 1) & 1u));
                        if (!ok) break;
                        fence_after();
                        const float factor = raise ? exp2_fast(ref - high) : 1.0f;
#pragma unroll
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_load32(o_addr + c, o);
                            tmem_wait_load(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                            tmem_store32(o_addr + c, o);
                        }
                        sum *= factor;
                    }
                    if (raise) ref = high;
                    const float base = ref == -INFINITY ? 0.0f : ref;
                    float add[4] = {0, 0, 0, 0};
                    uint32_t p[32];
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float u = exp2_fast(fmaf(__uint_as_float(s[c][e]), a.scale_log2, -base));
                            const float v = exp2_fast(fmaf(__uint_as_float(s[c][e + 1]), a.scale_log2, -base));
                            add[e & 2] += u;
                            add[(e & 2) + 1] += v;
                            p[c * 16 + e / 2] = pack2<TYPE>(u, v);
                        }
                    sum += (add[0] + add[1]) + (add[2] + add[3]);
                    __syncwarp();
                    tmem_store32(s_addr, p);
                    tmem_wait_store();
                }
                fence_before();
                mbar_arrive(&bar->p_ready[g][at & 1]);
            }
            if (!ok) break;
            done += blocks;
            ok = __all_sync(0xFFFFFFFFu, wait(&bar->pv_done[g][(done - 1) & 1], (uint32_t)((done - 1) >> 1) & 1u));
            if (!ok) break;
            fence_after();
            if (idle) continue;
            const float inverse = 1.0f / sum;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_load32(o_addr + c, o);
                tmem_wait_load(o);
                if (live) store_output<TYPE, HD>(t, plan, w, o, inverse, row, head, record, c);
                __syncwarp();
            }
            if (live && !w.item.direct) plan->part_ml[record] = make_float2(ref, sum);
            // The next item's first O overwrites this one after this group's next p_ready, so these loads are done.
            fence_before();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int TYPE, int HD>
cudaError_t launch(const TensorArgs &t, const CUtensorMap &map, cudaStream_t stream)
{
    auto kernel = tensor_attention_kernel<TYPE, HD>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void *>(kernel), Layout<HD>::kBytes);
    if (e != cudaSuccess) return e;
    return launch_overlapped(kernel, dim3(t.a.ctas), kThreads, Layout<HD>::kBytes, stream, t, map);
}

}  // namespace

bool tensor_attention_takes(int type, int head_dim)
{
    return (type == SATORI_F16 || type == SATORI_BF16) && (head_dim == 64 || head_dim == 128);
}

void tensor_plan_shape(int sm_count, PlanShape &shape)
{
    shape.tile_m = 2 * kTileRows;
    shape.block = kBlockKeys;
    shape.ctas = sm_count;
    shape.solo_m = kTileRows;
    // Hundreds of clocks: a block of a large tile, of a small one (HBM's share), and an item's start and end.
    shape.solo_cost = 10;
    shape.pair_cost = 14;
    shape.item_cost = 60;
    shape.slots_per_item = 2;
}

int tensor_record_rows() { return kTileRows; }

// cuTensorMapEncodeTiled through the runtime, so that the library loads where there is no driver.
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t make_page_map(CUtensorMap *map, void *memory, int type, int head_dim, int page_tokens, unsigned long long blocks)
{
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)page_tokens, (cuuint64_t)blocks};
    const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)head_dim * 2 * page_tokens};
    const cuuint32_t box[3] = {64, (cuuint32_t)std::min(page_tokens, kBlockKeys), 1}, ones[3] = {1, 1, 1};
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess || !f) return cudaErrorNotSupported;
    const CUresult r = reinterpret_cast<EncodeTiled>(f)(
        map, type == SATORI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, memory, dims,
        strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t launch_tensor_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream)
{
    TensorArgs t = {a, layer_block, 0, 0};
    t.wide_q = (uintptr_t)a.q % 16 == 0 && a.ldq % 8 == 0;
    t.wide_out = (uintptr_t)a.out % 16 == 0 && a.ldo * (a.out_f32 ? 4 : 2) % 16 == 0;
    if (a.type == SATORI_F16)
        return a.head_dim == 64 ? launch<SATORI_F16, 64>(t, map, stream) : launch<SATORI_F16, 128>(t, map, stream);
    return a.head_dim == 64 ? launch<SATORI_BF16, 64>(t, map, stream) : launch<SATORI_BF16, 128>(t, map, stream);
}

}  // namespace satori
