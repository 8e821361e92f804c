// batch_attn_tensor.cu -- attention of a batch over a paged 16-bit cache on the 5th-generation tensor cores, for
// heads of up to 128.  HD below is 64 or 128: columns from the head's own size on are zeros (the copies of K and V
// fill them in) and are neither read from q nor written.
//
// The same one pass over the keys as the FP32-unit kernel, as two matrix products per block of 64 keys:
// S = Q K^T and O += P V with P = 2^(s - m).  One CTA per SM works through its share of the plan's items:
//  * a thread of warp 16 loads the pages of a block's K and V with TMA (128-byte swizzle) into a ring of stages;
//  * one lane each of warps 17 and 18 issues the MMAs of a softmax group: S from shared memory (Q and K, both
//    K-major), O with P from tensor memory and V from shared memory as it lies (MN-major);
//  * warp 19 looks through the rows of V that not every row of the tile sees: it clears those behind the last key,
//    and takes infinities and NaN out of the others, which the rows that do see them get back at the end (a
//    weight of zero would turn them into NaN).  It also brings the queries of items of at most 24 rows (the usual
//    step of a request) while the items before are worked on, so that their first scores wait for nothing;
//  * warps 0-7 and 8-15 are two softmax groups, each with its own O and two S / P buffers in tensor memory; two
//    threads share a row, each with half of a block's keys and half of the output's columns.  A large tile
//    (129..256 rows) gives each group 128 of its rows and every K and V block serves both; a small one gives
//    each group every other block.  The scores of a group's next block are computed while it takes the
//    exponentials of this one.  Eight warps a group, not four: the exponentials are a chain of short steps, and
//    with two warps per scheduler it was idle two thirds of the time.
// The maximum that the exponentials refer to is raised only when it is exceeded by more than 2^8, so the
// accumulator in tensor memory is rescaled a few times per row, not at every block; P stays below 2^8 (beside fp16,
// whose small weights would lose bits, 2^15: see kLift) and the result does not depend on it.  P is rounded to the cache's type (half a step, as the operands already are);
// S, the sums and O are FP32.
//
// What bounds it: HBM and latencies for requests of their own (16 of exactly 4096 tokens, 28 heads of 128 over 4: 22 us a
// CTA, 20.8 at the rate of HBM, 35 us a call with start and merge).  For large tiles the softmax: a block of 256 rows and 64 keys takes 1750
// clocks with heads of 128 (64 requests behind 131072 tokens, 137 us) and 2000 with heads of 64, of which the
// exponentials' unit is busy 770 and the tensor pipe half; four warps a scheduler wait on chains of their own.  An item
// of one block takes about 6000 clocks, two at a time: 512 requests of one token 96 us.
#include "batch.cuh"
#include "common.cuh"

#include <algorithm>

namespace satori {

namespace {

constexpr int kTileRows = 128, kBlockKeys = 64;
constexpr int kSmallRows = 24;                 // rows of an item whose queries are brought ahead
constexpr int kGroupThreads = 2 * kTileRows, kThreads = 2 * kGroupThreads + 128;
// One pair of exponentials in four by a polynomial on the FP32 units: at 36 requests on 4096 shared keys and at 64 on
// 131072 about 6 % less time than with none, and no less with one in two or three.
constexpr int kEvery = 4;
constexpr float kLazy = 8.0f;                  // log2 of what a weight may exceed 1 by
// log2 of a factor of all weights and their sums.  fp16 ends at 2^16 above and keeps its 11 bits down to 2^-14: with the
// factor weights from 2^-21 of the reference on are rounded by half a step at most, and smaller ones by 2^-32.
template <int TYPE>
constexpr float kLift = TYPE == SATORI_F16 ? 7.0f : 0.0f;

template <int HD>
struct Layout {
    static constexpr int kQHalf = kTileRows * 128, kHalf = kBlockKeys * 128;       // rows of 64 columns
    static constexpr int kQTile = kQHalf * (HD / 64), kTile = kHalf * (HD / 64);   // Q; K or V
    static constexpr int kSmallHalf = kSmallRows * 128, kSmall = kSmallHalf * (HD / 64);       // Q brought ahead
    static constexpr int kStages = HD == 128 ? 9 : 20;
    static constexpr int kHeader = 4096;
    // header, 2 small Qs, 2 Q tiles, stages.  The MMAs read 128 rows from a small Q on, whatever lies behind it.
    static constexpr int kBytes = kHeader + 2 * kSmall + 2 * kQTile + kStages * kTile;
    static_assert((kHeader + 2 * kSmall) % 1024 == 0 && kSmallHalf % 1024 == 0, "swizzle");
    static constexpr int kOCol = 4 * kBlockKeys;                   // tensor memory: S / P buffers, then O
};

constexpr int kMaxStages = 20;
struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t s_full[2][2], p_ready[2][2];      // [group][buffer]: blocks in turn
    uint64_t q_ready[2], o_before[2], o_full[2];                   // o_before: all products but the item's last
    uint64_t edge_full[2], edge_clear[2], drained[2];
    uint64_t small_full[2], small_free[2];     // a small Q is there, or read
    uint32_t tmem;
    volatile int abort;
    float exchange[2][2][kTileRows];           // [group][half][row]: maximum, then sum
    // What warp 19 took out of V: the item (+ 1) that it concerns, and by column the first key, counted from the
    // first that not every row sees, with an infinity of either sign (with both: a NaN); 255: none.
    volatile int strange[2];
    volatile uint8_t first_strange[2][2][128];
    // Numbers and visible keys of the rows of the last small items.  Four: the second next is written when the scores
    // of this one are there, and the one in this one's place when those of the second next are, which follow this
    // one's weights in either group.
    int2 small_row[4][kSmallRows];
};
static_assert(sizeof(Barriers) <= 4096, "header");

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

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void *map, int c0, int c1, int c2, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
                 : "memory");
}

// All 64-column halves of a block of 64 tokens at token c1 of block c3 (the map of pages of 64 tokens and more).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, int token, int block, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(token), "r"(0), "r"(block), "r"(smem_u32(bar))
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
// 16 columns, waited for.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : SATORI_R8(v, 0), SATORI_R8(v, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::SATORI_W8(v, 0), SATORI_W8(v, 8), "r"(addr) : "memory");
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

// NaN if any of them is.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// 2^x on the FP32 units, two at a time, for part of the weights: the special function unit takes 8 clocks for a
// warp's exponentials and is the scarcer one.  x = n + f with n the nearest integer (left in the low bits of
// x + 1.5 2^23) and 2^f by a polynomial: the minimax fits on |f| <= 1/2 of degree 3 (relative error 7.5e-5,
// 1/26 of bf16's half step) and 4 (2.6e-6, for fp16); n goes into the exponent.  x below -126 counts as -126, and so
// does a NaN, which the row's other weights and its sum then carry (see the maximum).
template <int TYPE>
__device__ __forceinline__ float2 exp2_poly(float2 x)
{
    const float2 magic = make_float2(12582912.0f, 12582912.0f), minus = make_float2(-1.0f, -1.0f);
    x.x = fmaxf(x.x, -126.0f);
    x.y = fmaxf(x.y, -126.0f);
    const float2 t = __fadd2_rn(x, magic);
    const float2 n = __fadd2_rn(t, make_float2(-12582912.0f, -12582912.0f));
    const float2 f = __ffma2_rn(n, minus, x);
    float2 p;
    auto pair = [](float v) { return make_float2(v, v); };
    if (TYPE == SATORI_BF16) {
        p = __ffma2_rn(pair(0.05517165765016593f), f, pair(0.24261112131938758f));
        p = __ffma2_rn(p, f, pair(0.6932609875663172f));
        p = __ffma2_rn(p, f, pair(0.9999280736469822f));
    } else {
        p = __ffma2_rn(pair(0.009570100592456837f), f, pair(0.05591786021593906f));
        p = __ffma2_rn(p, f, pair(0.24024744860429012f));
        p = __ffma2_rn(p, f, pair(0.6931218147559814f));
        p = __ffma2_rn(p, f, pair(0.9999992614359087f));
    }
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
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

// Named barriers of the two warps that share 32 rows.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool mine)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, 64, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(any) : "r"((uint32_t)mine), "r"(id) : "memory");
    return any != 0;
}

// Weights of 32 scores, packed in pairs, and their sum.  Every EVERY-th pair takes the polynomial
// (0: none).
template <int TYPE, int EVERY>
__device__ __forceinline__ float block_weights(const uint32_t (&s)[32], float scale, float base, uint32_t (&p)[16])
{
    const float2 scale2 = make_float2(scale, scale), minus_base = make_float2(-base, -base);
    float2 add[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, minus_base);
        float2 w;
        if (EVERY > 0 && (e / 2) % (EVERY > 0 ? EVERY : 1) == 0)
            w = exp2_poly<TYPE>(x);
        else
            w = make_float2(exp2_fast(x.x), exp2_fast(x.y));
        add[e / 2 & 1] = __fadd2_rn(add[e / 2 & 1], w);
        p[e / 2] = pack2<TYPE>(w.x, w.y);
    }
    const float2 sum = __fadd2_rn(add[0], add[1]);
    return sum.x + sum.y;
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
    int flip;            // items in turn give their first block to group 0 and 1, so that two short ones run at once
    // Blocks of each softmax group, and how many blocks ahead of O the scores run.  An item's loads are in the
    // order of use: the leading blocks' K, then V and the next K in turn.
    __device__ __forceinline__ int blocks(int g) const { return pair ? item.blocks : (item.blocks + 1 - (g ^ flip)) / 2; }
    __device__ __forceinline__ bool takes(int g, int j) const { return pair || ((j ^ flip) & 1) == g; }
    __device__ __forceinline__ int block(int g, int k) const { return item.block0 + (pair ? k : 2 * k + (g ^ flip)); }
    __device__ __forceinline__ int lead() const { return min(item.blocks, pair ? 2 : 4); }
    __device__ __forceinline__ bool small() const { return item.m <= kSmallRows; }
    // Keys of the tile that every row of it sees.
    __device__ __forceinline__ int seen_by_all(const DevPlan *plan, int group) const
    {
        if (item.start < 0 || item.m0 % group + item.m <= group) return item.keys;
        const int2 row = __ldg(reinterpret_cast<const int2 *>(plan_array<PlanRow>(plan, plan->seg_rows) + item.row_off) + item.m0 / group);
        return row.y + 1 - item.start;
    }
    // The item's first block with keys that not every row sees, or with none; item.blocks or more: no such block.
    __device__ __forceinline__ int edge(int seen) const { return max(0, seen - item.block0 * kBlockKeys) / kBlockKeys; }
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
    w.flip = i & 1;
    return w;
}

// The number of a segment's row and how many of its keys the row sees.
__device__ __forceinline__ int2 find_row(const DevPlan *plan, const Work &w, int group, int m)
{
    int2 own = __ldg(reinterpret_cast<const int2 *>(plan_array<PlanRow>(plan, plan->seg_rows) + w.item.row_off) + m / group);
    own.y = w.item.start >= 0 ? own.y + 1 - w.item.start : w.item.keys;
    return own;
}

// 16 bytes from any address of 2-byte elements.
__device__ __noinline__ uint4 load_unaligned(const void *src)
{
    const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
    return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                      h[6] | (uint32_t)h[7] << 16);
}

// Whether any of 8 values is infinite or NaN: an exponent of ones carries into the sign's place.
template <int TYPE>
__device__ __forceinline__ bool not_finite(uint4 v)
{
    constexpr uint32_t kExponent = TYPE == SATORI_BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = TYPE == SATORI_BF16 ? 0x00800080u : 0x04000400u;
    return (((v.x & kExponent) + kOne) | ((v.y & kExponent) + kOne) | ((v.z & kExponent) + kOne) | ((v.w & kExponent) + kOne)) & 0x80008000u;
}

// Notes for group g the infinities and NaN in rows lo .. have - 1 of a block of V, whose row 0 is `key` keys behind
// the first that not every row sees, and (unless they are to be noted for the other group too) sets them to zero.
// A tile's rows stand for at most 256 tokens, so a key that one of them sees and another does not is at most the
// 255th; a later row of the block is seen by none.  Called by a whole warp; each lane has columns of its own.
template <int TYPE, int HD>
__device__ __noinline__ void take_out(Barriers *bar, int g, int tag, uint8_t *v, int lo, int have, int key, bool again)
{
    const int lane = threadIdx.x & 31;
    const bool fresh = bar->strange[g] != tag;
    __syncwarp();
    for (int c = lane; c < HD; c += 32) {
        int first[2] = {255, 255};
        if (!fresh) {
            first[0] = bar->first_strange[g][0][c];
            first[1] = bar->first_strange[g][1][c];
        }
        for (int r = lo; r < have; ++r) {
            uint16_t *at = reinterpret_cast<uint16_t *>(v + c / 64 * Layout<HD>::kHalf + r * 128 + ((((c % 64) / 8) ^ (r & 7)) * 16) + c % 8 * 2);
            const uint32_t x = *at, exponent = TYPE == SATORI_BF16 ? 0x7F80u : 0x7C00u;
            if ((x & exponent) != exponent) continue;
            const bool nan = x & ~exponent & 0x7FFFu;
            if (nan || !(x & 0x8000u)) first[0] = min(first[0], key + r);
            if (nan || (x & 0x8000u)) first[1] = min(first[1], key + r);
            if (!again) *at = 0;
        }
        bar->first_strange[g][0][c] = (uint8_t)first[0];
        bar->first_strange[g][1][c] = (uint8_t)first[1];
    }
    if (lane == 0) bar->strange[g] = tag;
    __syncwarp();
}

// Adds what take_out noted to `n` columns from c on of a row that sees `keys` of the keys that not every row sees,
// where this thread has just stored them: floats `step` apart for every 4, or outputs.
template <typename T>
__device__ __noinline__ void put_back(const Barriers *bar, int g, int keys, int c, int n, T *at, int step)
{
    for (int e = 0; e < n; ++e) {
        T *to = at + e / 4 * step + e % 4;
        float v = (float)*to;
        if (keys > bar->first_strange[g][0][c + e]) v += INFINITY;
        if (keys > bar->first_strange[g][1][c + e]) v -= INFINITY;
        *to = (T)v;
    }
}

// 32 columns of a row's accumulator: its share of the partial record, or of an output with 16-byte accesses.
template <int TYPE>
__device__ __forceinline__ void store_output(const BatchAttn &a, const DevPlan *plan, const Work &w, uint32_t *o,
                                             float inverse, int row, int head, long long record, int c)
{
    if (!w.item.direct) {
        // [column / 4][row]: the warp's rows are neighbours.
        const int r = (int)(record % kTileRows);
        uint4 *dst = reinterpret_cast<uint4 *>(plan->part_o) + (record - r) * (a.head_dim / 4) + (c / 4) * kTileRows + r;
#pragma unroll
        for (int e = 0; e < 32; e += 4)
            if (c + e < a.head_dim) dst[e / 4 * kTileRows] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        return;
    }
    const long long to = (long long)row * a.ldo + (long long)head * a.head_dim + c;
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inverse);
    if (a.out_f32) {
        uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<float *>(a.out) + to);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
            if (c + e < a.head_dim) dst[e / 4] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    } else {
        uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<typename Elem<TYPE>::type *>(a.out) + to);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
            uint4 v;
            v.x = pack2<TYPE>(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
            v.y = pack2<TYPE>(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
            v.z = pack2<TYPE>(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]));
            v.w = pack2<TYPE>(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7]));
            if (c + e < a.head_dim) dst[e / 8] = v;
        }
    }
}

// Up to 16 columns of an output row at any address.
template <int TYPE>
__device__ __noinline__ void store_anywhere(const BatchAttn &a, const uint32_t *o, float inverse, long long to, int n)
{
    for (int e = 0; e < min(16, n); ++e) {
        const float v = __uint_as_float(o[e]) * inverse;
        if (a.out_f32)
            reinterpret_cast<float *>(a.out)[to + e] = v;
        else
            reinterpret_cast<typename Elem<TYPE>::type *>(a.out)[to + e] = Elem<TYPE>::from_float(v);
    }
}

// An item's loads, in the order of use, by one thread.  What it does for a load is on the way of everything else
// (with the page numbers fetched in line by a lane per box it took 1170 clocks a load, and the kernel waited
// for nothing else), so the page numbers are fetched a step ahead and a whole block of 64-token pages is one copy.
template <int HD>
struct Loads {
    const TensorArgs &t;
    const CUtensorMap &map;
    Barriers *bar;
    uint32_t stages;
    const int *pages;
    int keys, first_block;

    // PER: pages of a block.
    template <int PER, typename Wait>
    __device__ __forceinline__ bool run(const Work &w, Ring<Layout<HD>::kStages> &ring, int &units, Wait &wait) const
    {
        typedef Layout<HD> L;
        constexpr int kBox = kBlockKeys / PER;
        const int shift = __ffs(t.a.page_tokens) - 1, mask = t.a.page_tokens - 1, n = w.item.blocks, lead = w.lead();
        const int key0 = w.item.block0 * kBlockKeys, page_blocks = 2 * t.a.kv_heads;
        const int last_boxes = (min(kBlockKeys, keys - key0 - (n - 1) * kBlockKeys) + kBox - 1) / kBox;
        auto fetch = [&](int j, int (&id)[PER]) {
#pragma unroll
            for (int b = 0; b < PER; ++b) {
                const int key = key0 + j * kBlockKeys + b * kBox;
                if (key < keys) id[b] = __ldg(pages + (key >> shift));
            }
        };
        auto issue = [&](int j, int kv, const int (&id)[PER]) -> bool {
            uint64_t *full = &bar->full[ring.stage];
            if (!wait(&bar->empty[ring.stage], ring.parity ^ 1u)) return false;
            const uint32_t to = stages + ring.stage * L::kTile;
            const int boxes = j == n - 1 ? last_boxes : PER, block0 = first_block + kv * t.a.kv_heads;
            mbar_expect_tx(full, (uint32_t)(boxes * kBox * HD * 2));
            if (PER == 1 && t.a.head_dim % 64 == 0) {
                tma_load_4d(to, &map, (key0 + j * kBlockKeys) & mask, block0 + id[0] * page_blocks, full);
            } else {
#pragma unroll
                for (int b = 0; b < PER; ++b)
                    if (b < boxes)
#pragma unroll
                        for (int half = 0; half < HD / 64; ++half)
                            tma_load_3d(to + half * L::kHalf + b * kBox * 128, &map, half * 64,
                                        PER == 1 ? (key0 + j * kBlockKeys) & mask : 0, block0 + id[b] * page_blocks, full);
            }
            ring.next();
            ++units;
            return true;
        };
        int k_id[PER], v_id[PER];
#pragma unroll
        for (int b = 0; b < PER; ++b) k_id[b] = v_id[b] = 0;
        fetch(0, k_id);
        fetch(0, v_id);
        for (int j = 0; j < lead; ++j) {
            int next[PER];
#pragma unroll
            for (int b = 0; b < PER; ++b) next[b] = 0;
            if (j + 1 < n) fetch(j + 1, next);
            if (!issue(j, 0, k_id)) return false;
#pragma unroll
            for (int b = 0; b < PER; ++b) k_id[b] = next[b];
        }
        for (int j = 0; j < n; ++j) {
            int next_v[PER], next_k[PER];
#pragma unroll
            for (int b = 0; b < PER; ++b) next_v[b] = next_k[b] = 0;
            if (j + 1 < n) fetch(j + 1, next_v);
            if (j + lead + 1 < n) fetch(j + lead + 1, next_k);
            if (!issue(j, 1, v_id)) return false;
            if (j + lead < n && !issue(j + lead, 0, k_id)) return false;
#pragma unroll
            for (int b = 0; b < PER; ++b) {
                v_id[b] = next_v[b];
                k_id[b] = next_k[b];
            }
        }
        return true;
    }
};

template <int TYPE, int HD>
__global__ void __launch_bounds__(kThreads, 1) tensor_attention_kernel(const TensorArgs t, const __grid_constant__ CUtensorMap map)
{
    typedef Layout<HD> L;
    typedef typename Elem<TYPE>::type T;
    constexpr int NS = L::kStages;
    const BatchAttn &a = t.a;
    extern __shared__ __align__(1024) uint8_t smem[];
    Barriers *bar = reinterpret_cast<Barriers *>(smem);
    uint8_t *small_q = smem + L::kHeader, *q_tiles = small_q + 2 * L::kSmall, *stages = q_tiles + 2 * L::kQTile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (smem_u32(smem) & 1023u) {              // the swizzle needs it; dynamic shared memory starts there
        if (tid == 0) atomicOr(a.err, kDevErrTimeout);
        return;
    }
    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar->full[s], 1);
            mbar_init(&bar->empty[s], 2);
        }
        for (int g = 0; g < 2; ++g) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bar->s_full[g][b], 1);
                mbar_init(&bar->p_ready[g][b], kGroupThreads);
            }
            mbar_init(&bar->q_ready[g], kGroupThreads);
            mbar_init(&bar->o_before[g], 1);
            mbar_init(&bar->o_full[g], 1);
            mbar_init(&bar->edge_full[g], 1);
            mbar_init(&bar->edge_clear[g], 32);
            mbar_init(&bar->drained[g], 1);
            mbar_init(&bar->small_full[g], 1);
            mbar_init(&bar->small_free[g], 2);
        }
        bar->abort = bar->strange[0] = bar->strange[1] = 0;
        fence_mbar_init();
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar->tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp == 16 && lane == 0) prefetch_tensormap(&map);
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

    if (warp == 16) {
        // ---- loads, by one thread
        if (elect_one()) {
            Ring<NS> ring;
            int units = 0;
            bool ok = true;
            for (int i = first; i < last && ok; ++i) {
                const Work w = load_work(plan, i);
                const int *pages = plan_array<int>(plan, plan->pages) + w.item.page_off;
                const Loads<HD> loads = {t, map, bar, smem_u32(stages), pages, w.item.keys, t.layer_block + w.item.kv_head};
                ok = a.page_tokens >= kBlockKeys ? loads.template run<1>(w, ring, units, wait)
                     : a.page_tokens == 32       ? loads.template run<2>(w, ring, units, wait)
                                                 : loads.template run<4>(w, ring, units, wait);
            }
            if (!ok)      // the copies in flight land before the CTA may end
                for (int u = max(0, units - NS); u < units; ++u) mbar_wait_bounded(&bar->full[u % NS], (uint32_t)((u / NS) & 1));
        }
        __syncwarp();
    } else if (warp == 19) {
        // ---- V at the edge of what the rows see, and small Qs ahead
        Ring<NS> ring;
        uint32_t phase = 0;                            // bit g: edge_full[g]
        bool ok = true;
        int smalls = 0;                                // small items so far
        auto bring = [&](int i) -> bool {
            if (i >= last) return true;
            const Work w = load_work(plan, i);
            if (!w.small()) return true;
            constexpr int PER_ROW = HD / 8, ROWS = 32 / PER_ROW, BATCH = 6, BATCHES = kSmallRows / (ROWS * BATCH);
            static_assert(BATCHES * ROWS * BATCH == kSmallRows, "rows");
            const int b = smalls & 1, m = w.item.m0 + lane;
            const int2 own = lane < w.item.m ? find_row(plan, w, a.group, m) : make_int2(0, 0);
            const int row = own.x;
            const int q_head = (w.item.kv_head * a.group + m % a.group) * a.head_dim, c = lane % PER_ROW;
            uint8_t *q_tile = small_q + b * L::kSmall;
            const bool free = __all_sync(0xFFFFFFFFu, wait(&bar->small_free[b], (uint32_t)((smalls >> 1) & 1) ^ 1u));
            if (!free) return false;
            if (lane < kSmallRows) bar->small_row[smalls & 3][lane] = own;
#pragma unroll
            for (int k = 0; k < BATCHES; ++k) {
                if (k * BATCH * ROWS >= w.item.m) break;
                uint4 v[BATCH];
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    const int from = (k * BATCH + e) * ROWS + lane / PER_ROW;
                    const int r_from = __shfl_sync(0xFFFFFFFFu, row, from), h_from = __shfl_sync(0xFFFFFFFFu, q_head, from);
                    const T *src = reinterpret_cast<const T *>(a.q) + (long long)r_from * a.ldq + h_from + c * 8;
                    v[e] = make_uint4(0, 0, 0, 0);
                    if (from < w.item.m && c * 8 < a.head_dim) v[e] = t.wide_q ? __ldg(reinterpret_cast<const uint4 *>(src)) : load_unaligned(src);
                }
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    const int from = (k * BATCH + e) * ROWS + lane / PER_ROW;
                    *reinterpret_cast<uint4 *>(q_tile + (c / 8) * L::kSmallHalf + from * 128 + (((c & 7) ^ (from & 7)) * 16)) = v[e];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->small_full[b]);
            ++smalls;
            return true;
        };
        ok = bring(first) && bring(first + 1);
        for (int i = first; i < last && ok; ++i) {
            const Work w = load_work(plan, i);
            const int n = w.item.blocks, lead = w.lead(), seen = w.seen_by_all(plan, a.group);
            int at = 0;                                // the item's loads passed
            for (int j = w.edge(seen); j < n; ++j) {
                const int unit = lead + j + min(j, n - lead);
                ring.advance(unit - at);
                at = unit;
                // The MMA warps that use the block have seen the load arrive, and wait: the stage keeps its contents,
                // and the groups are done with the last item's findings.
                for (int g = 0; g < 2 && ok; ++g) {
                    if (!w.takes(g, j)) continue;
                    ok = __all_sync(0xFFFFFFFFu, wait(&bar->edge_full[g], phase >> g & 1u));
                    phase ^= 1u << g;
                }
                if (!ok) break;
                const int key0 = (w.item.block0 + j) * kBlockKeys, have = min(kBlockKeys, w.item.keys - key0);
                const int lo = min(have, max(0, seen - key0));
                uint8_t *v = stages + (size_t)ring.stage * L::kTile;
                bool strange = false;
                for (int c = lane; c < (have - lo) * 8; c += 32)
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h)
                        strange |= not_finite<TYPE>(*reinterpret_cast<const uint4 *>(v + h * L::kHalf + lo * 128 + c * 16));
                if (__any_sync(0xFFFFFFFFu, strange)) {
                    for (int g = 0; g < 2; ++g)
                        if (w.takes(g, j)) take_out<TYPE, HD>(bar, g, i + 1, v, lo, have, key0 - seen, w.pair && g == 0);
                }
                for (int c = have * 8 + lane; c < kBlockKeys * 8; c += 32)
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h) *reinterpret_cast<uint4 *>(v + h * L::kHalf + c * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                for (int g = 0; g < 2; ++g)
                    if (w.takes(g, j)) mbar_arrive(&bar->edge_clear[g]);
            }
            ring.advance(2 * n - at);
            ok = ok && bring(i + 2);                   // (its Q takes this one's place when the scores are there)
        }
    } else if (warp == 17 || warp == 18) {
        // ---- matrix products of group g
        const int g = warp - 17;
        if (elect_one()) {
            constexpr uint32_t kFormat = TYPE == SATORI_BF16 ? 1u : 0u;
            // FP32 accumulator, A and B of the cache's type, M = 128; S: N = 64, both K-major; O: N = HD, B MN-major.
            constexpr uint32_t kBase = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(kTileRows >> 4) << 24);
            constexpr uint32_t kDescS = kBase | ((uint32_t)(kBlockKeys >> 3) << 17);
            constexpr uint32_t kDescO = kBase | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
            const uint32_t q_low = desc_low(smem_u32(q_tiles) + g * L::kQTile, 16), k_low = desc_low(smem_u32(stages), 16);
            const uint32_t v_low = desc_low(smem_u32(stages), L::kHalf), s_col = tmem + g * 2 * kBlockKeys;
            const uint32_t o_col = tmem + L::kOCol + g * HD;
            // Both groups pass every load in order, and a stage is loaded again when both have released it: so
            // the parity that a group waits for is never a round ahead of or behind the stage's.
            Ring<NS> ring;
            uint32_t q_phase = 0, edge_phase = 0;
            int done = 0, smalls = 0;                  // this group's blocks, and the small items, so far
            bool ok = true, issued = false;
            for (int i = first; i < last && ok; ++i) {
                const Work w = load_work(plan, i);
                const int n = w.blocks(g), all = w.item.blocks, lead = w.lead(), seen = w.seen_by_all(plan, a.group);
                const int edge = w.edge(seen), b = smalls & 1;
                const bool small = w.small();
                uint32_t q = q_low;
                const uint32_t q_half = small ? L::kSmallHalf >> 4 : L::kQHalf >> 4;
                if (small) {
                    q = desc_low(smem_u32(small_q) + b * L::kSmall, 16);
                    // (A group without a block waits too: its next wait is for the next turn's parity.)
                    ok = wait(&bar->small_full[b], (uint32_t)(smalls >> 1) & 1u);
                    if (n == 0)
                        mbar_arrive(&bar->small_free[b]);
                    else
                        issued = issued || ok;
                    ++smalls;
                } else if (n > 0) {
                    ok = wait(&bar->q_ready[g], q_phase);
                    q_phase ^= 1u;
                    issued = issued || ok;
                }
                auto mine = [&](int j) { return w.takes(g, j); };
                auto index = [&](int j) { return w.pair ? j : j >> 1; };
                int held = -1;                         // a stage of V to release after the next scores
                auto release_held = [&] {
                    if (held >= 0) commit(&bar->empty[held]);
                    held = -1;
                };
                // S = Q K^T of block j, or K of the other group's block.
                auto scores = [&](int j) -> bool {
                    if (!wait(&bar->full[ring.stage], ring.parity)) return false;
                    if (mine(j)) {
                        const int at = done + index(j);
                        fence_after();
                        const uint32_t d = s_col + (at & 1) * kBlockKeys, kd = k_low + ring.stage * (L::kTile >> 4);
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks)
                            mma_ss(d, q + (ks / 4) * q_half + (ks % 4) * 2,
                                   kd + (ks / 4) * (L::kHalf >> 4) + (ks % 4) * 2, kDescS, ks > 0);
                        commit(&bar->s_full[g][at & 1]);
                        if (small && index(j) == n - 1) commit(&bar->small_free[b]);
                        release_held();
                        commit(&bar->empty[ring.stage]);
                    } else {
                        mbar_arrive(&bar->empty[ring.stage]);
                    }
                    ring.next();
                    return true;
                };
                // O += P V of block j, once P is there.
                auto values = [&](int j) -> bool {
                    if (!wait(&bar->full[ring.stage], ring.parity)) return false;
                    if (mine(j)) {
                        const int k = index(j), at = done + k;
                        if (j >= edge) {
                            // What warp 19 takes out is noted when the group is done with the last item's notes.
                            if (small && seen < w.item.keys && !wait(&bar->p_ready[g][at & 1], (uint32_t)(at >> 1) & 1u)) return false;
                            mbar_arrive(&bar->edge_full[g]);
                            if (!wait(&bar->edge_clear[g], edge_phase)) return false;
                            edge_phase ^= 1u;
                        }
                        if (!wait(&bar->p_ready[g][at & 1], (uint32_t)(at >> 1) & 1u)) return false;
                        fence_after();
                        const uint32_t p = s_col + (at & 1) * kBlockKeys, vd = v_low + ring.stage * (L::kTile >> 4);
#pragma unroll
                        for (int ks = 0; ks < kBlockKeys / 16; ++ks)
                            mma_ts(o_col, p + ks * 8, vd + ks * (2048 >> 4), kDescO, ks > 0 || k > 0);
                        // The next scores in this buffer follow O, which has read its weights; with them due, the
                        // stage is released behind them.
                        held = ring.stage;
                        if (k + 2 >= n) {
                            commit(k + 1 < n ? &bar->o_before[g] : &bar->o_full[g]);
                            release_held();
                        }
                    } else {
                        mbar_arrive(&bar->empty[ring.stage]);
                    }
                    ring.next();
                    return true;
                };
                for (int j = 0; j < lead && ok; ++j) ok = scores(j);
                for (int j = 0; j < all && ok; ++j) {
                    ok = values(j);
                    if (ok && j + lead < all) ok = scores(j + lead);
                }
                done += n;
            }
            // The issued MMAs finish before the tensor memory is freed.
            if (issued) {
                commit(&bar->drained[g]);
                mbar_wait_bounded(&bar->drained[g], 0);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: the threads (half 0 and 1, r) of group g own tile row r (and tensor memory lane r).  Their
        // waits are not left on an expired one: the two warps of a row meet at named barriers, so each goes
        // on to the end, where every further wait returns at once.
        const int g = warp >> 3, half = warp >> 2 & 1, quad = warp & 3, r = quad * 32 + lane;
        const int pair_id = 1 + g * 4 + quad;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t o_addr = lanes + L::kOCol + g * HD + half * (HD / 2);
        uint8_t *q_tile = q_tiles + g * L::kQTile;
        int done = 0, smalls = 0;              // this group's blocks, and the small items, so far
        uint32_t before_phase = 0, full_phase = 0;
        for (int i = first; i < last; ++i) {
            const Work w = load_work(plan, i);
            const int blocks = w.blocks(g);
            const int m = (w.pair ? g * kTileRows : 0) + r;
            const bool live = m < w.item.m;
            const long long record = (long long)(w.item.slot + g) * kTileRows + r;
            // The row's number and the keys it sees.  A small item's are read behind its first scores, which came after
            // warp 19 had written them: a wait of the group's own for them might come two turns late, when its
            // parity is that of a turn still to come.
            int2 own = make_int2(0, 0);
            const int small = smalls & 3;
            if (w.small())
                ++smalls;
            else if (live)
                own = find_row(plan, w, a.group, w.item.m0 + m);
            if (blocks == 0) {                 // a small tile's only block is the other group's
                if (live && half == 0 && !w.item.direct) plan->part_ml[record] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            const int head = w.item.kv_head * a.group + (w.item.m0 + m) % a.group;
            // Q rows into shared memory (each half 16 of the warp pair's 32), K-major with the 128-byte swizzle:
            // 16-byte chunk c of row r lies at chunk c ^ (r % 8).  Rows behind the tile keep what was there: their
            // lanes of S and O are never read.  All loads are in flight before the first store.
            const int warp_rows = min(32, w.item.m - (m - lane));          // live rows of the warp pair
            if (half * 16 < warp_rows && !w.small()) {
                constexpr int PER_ROW = HD / 8, ROWS = 32 / PER_ROW, STEPS = 16 / ROWS;
                const int c = lane % PER_ROW, mine = half * 16 + lane / PER_ROW, q_head = head * a.head_dim;
                uint4 v[STEPS];
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const int from = mine + k * ROWS;
                    const int r_from = __shfl_sync(0xFFFFFFFFu, own.x, from), h_from = __shfl_sync(0xFFFFFFFFu, q_head, from);
                    const T *src = reinterpret_cast<const T *>(a.q) + (long long)r_from * a.ldq + h_from + c * 8;
                    v[k] = make_uint4(0, 0, 0, 0);
                    if (from < warp_rows && c * 8 < a.head_dim) v[k] = t.wide_q ? __ldg(reinterpret_cast<const uint4 *>(src)) : load_unaligned(src);
                }
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const int from = mine + k * ROWS, rr = quad * 32 + from;
                    if (from < warp_rows)
                        *reinterpret_cast<uint4 *>(q_tile + (c / 8) * L::kQHalf + rr * 128 + (((c & 7) ^ (rr & 7)) * 16)) = v[k];
                }
            }
            if (!w.small()) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&bar->q_ready[g]);
            }

            const bool idle = warp_rows <= 0;  // all of the warp pair's rows are behind the tile
            float ref = -INFINITY, sum = 0;    // ref: the maximum (log2 units) that the weights refer to
            for (int k = 0; k < blocks; ++k) {
                const int block = w.block(g, k), at = done + k;
                const uint32_t s_addr = lanes + (g * 2 + (at & 1)) * kBlockKeys;
                wait(&bar->s_full[g][at & 1], (uint32_t)(at >> 1) & 1u);
                if (!idle) {
                    __syncwarp();
                    fence_after();
                    if (k == 0 && live && w.small()) own = bar->small_row[small][r];
                    const int see = own.y - block * kBlockKeys - half * 32;        // keys of this half that the row sees
                    uint32_t s[32];
                    tmem_load32(s_addr + half * 32, s);
                    tmem_wait_load(s);
                    const bool masked = __any_sync(0xFFFFFFFFu, see < 32);
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= see) s[e] = 0xFF800000u;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; e += 2) top[e / 2 & 3] = max3(top[e / 2 & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                    // A score that is NaN or plus infinity makes the row NaN: the maximum is NaN then, which is above
                    // no bound and below none, and so are the weights that refer to it and their sum from there on.
                    float high = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
                    // (The barrier also keeps one half's weights from the scores that the other has yet to read.)
                    if (pair_any(pair_id, !(high <= ref + kLazy))) {
                        bar->exchange[g][half][r] = high;
                        pair_sync(pair_id);
                        high = max3(high, bar->exchange[g][half ^ 1][r], high);
                        if (high == INFINITY) high = NAN;
                        const bool raise = !(high <= ref + kLazy);
                        if (k > 0) {
                            // The last block's product may still be adding to O.  The next block's scores follow it.
                            if (k + 1 < blocks)
                                wait(&bar->s_full[g][(at + 1) & 1], (uint32_t)((at + 1) >> 1) & 1u);
                            else
                                wait(&bar->o_before[g], before_phase);
                            __syncwarp();
                            fence_after();
                            const float factor = raise ? exp2_fast(ref - high) : 1.0f;
#pragma unroll 1
                            for (int c = 0; c < HD / 2; c += 16) {
                                uint32_t o[16];
                                tmem_load16(o_addr + c, o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                                tmem_store16(o_addr + c, o);
                            }
                            sum *= factor;
                        }
                        if (raise) ref = high;
                    }
                    const float base = (ref == -INFINITY ? 0.0f : ref) - kLift<TYPE>;
                    uint32_t p[16];
                    // A masked key's weight is exactly zero, which the polynomial cannot give.
                    sum += masked ? block_weights<TYPE, 0>(s, a.scale_log2, base, p)
                                  : block_weights<TYPE, kEvery>(s, a.scale_log2, base, p);
                    __syncwarp();
                    tmem_store16(s_addr + half * 16, p);
                    tmem_wait_store();
                }
                fence_before();
                mbar_arrive(&bar->p_ready[g][at & 1]);
            }
            done += blocks;
            if (blocks > 1) before_phase ^= 1u;
            wait(&bar->o_full[g], full_phase);
            full_phase ^= 1u;
            if (idle) continue;
            bar->exchange[g][half][r] = sum;
            pair_sync(pair_id);
            sum += bar->exchange[g][half ^ 1][r];
            __syncwarp();
            fence_after();
            const float inverse = 1.0f / sum;
            const bool strange = bar->strange[g] == i + 1;
            const int c0 = half * (HD / 2);
            const long long to = (long long)own.x * a.ldo + (long long)head * a.head_dim + c0;
            // (Rolled, like the rescaling above: this code runs once an item, and fetching it took most of its time.)
            if (w.item.direct && !t.wide_out) {
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 16) {
                    uint32_t o[16];
                    tmem_load16(o_addr + c, o);
                    if (live) store_anywhere<TYPE>(a, o, inverse, to + c, a.head_dim - c0 - c);
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 32) {
                    uint32_t o[32];
                    tmem_load32(o_addr + c, o);
                    tmem_wait_load(o);
                    if (live) store_output<TYPE>(a, plan, w, o, inverse, own.x, head, record, c0 + c);
                    __syncwarp();
                }
            }
            if (strange && live) {
                const int keys = own.y - w.seen_by_all(plan, a.group), n = min(HD / 2, a.head_dim - c0);
                if (!w.item.direct)
                    put_back(bar, g, keys, c0, n, plan->part_o + ((record - r) * a.head_dim + c0 * kTileRows + r * 4), kTileRows * 4);
                else if (a.out_f32)
                    put_back(bar, g, keys, c0, n, reinterpret_cast<float *>(a.out) + to, 4);
                else
                    put_back(bar, g, keys, c0, n, reinterpret_cast<T *>(a.out) + to, 4);
            }
            if (live && half == 0 && !w.item.direct) plan->part_ml[record] = make_float2(ref, sum);
            // The next item's first O overwrites this one after this group's next p_ready, so these loads are done.
            // The other half has read this sum before either writes the exchange again (both pass pair_any first).
            fence_before();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
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
    return (type == SATORI_F16 || type == SATORI_BF16) && head_dim <= 128;
}

void tensor_plan_shape(int sm_count, PlanShape &shape)
{
    shape.tile_m = 2 * kTileRows;
    shape.block = kBlockKeys;
    shape.ctas = sm_count;
    shape.solo_m = kTileRows;
    // About 120 clocks each: a block of a small tile (HBM's share), of a large one, an item's start and end, and the
    // shortest item, which is a chain of latencies.  An item at 60 leaves CTAs with few items behind those with many:
    // 512 requests of 100 tokens behind 2048 then take 211 us and not 157, 64 of 1000 over 32 KV heads 101 and not 82;
    // a large block at 20 costs 64 requests behind 32k tokens 73 and not 67 us.
    shape.solo_cost = 10;
    shape.pair_cost = 16;
    shape.item_cost = 30;
    shape.least_cost = 50;
    shape.slots_per_item = 2;
}

int tensor_record_rows() { return kTileRows; }

// cuTensorMapEncodeTiled through the runtime, so that the library loads where there is no driver.
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t make_page_map(CUtensorMap *map, void *memory, int type, int head_dim, int page_tokens, unsigned long long blocks)
{
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess || !f) return cudaErrorNotSupported;
    const CUtensorMapDataType kind = type == SATORI_F16   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : type == SATORI_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint32_t size = type == SATORI_F32 ? 4 : 2, columns = 128 / size;      // columns of a 128-byte tile row
    const cuuint64_t row = (cuuint64_t)head_dim * size, block = row * page_tokens;
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    CUresult r;
    if (page_tokens >= kBlockKeys && head_dim % columns == 0) {        // [block][part][token][columns]: a box is a block of keys, part by part
        const cuuint64_t dims[4] = {columns, (cuuint64_t)page_tokens, (cuuint64_t)head_dim / columns, (cuuint64_t)blocks};
        const cuuint64_t strides[3] = {row, 128, block};
        const cuuint32_t box[4] = {columns, kBlockKeys, (cuuint32_t)head_dim / columns, 1};
        r = reinterpret_cast<EncodeTiled>(f)(map, kind, 4, memory, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {                               // [block][token][dim]: a box is 128 bytes (zeros behind the head) of a page's rows
        const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)page_tokens, (cuuint64_t)blocks}, strides[2] = {row, block};
        const cuuint32_t box[3] = {columns, std::min<cuuint32_t>(page_tokens, kBlockKeys), 1};
        r = reinterpret_cast<EncodeTiled>(f)(map, kind, 3, memory, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t launch_tensor_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream)
{
    TensorArgs t = {a, layer_block, 0, 0};
    t.wide_q = (uintptr_t)a.q % 16 == 0 && a.ldq % 8 == 0;
    t.wide_out = (uintptr_t)a.out % 16 == 0 && a.ldo * (a.out_f32 ? 4 : 2) % 16 == 0;
    if (a.type == SATORI_F16)
        return a.head_dim <= 64 ? launch<SATORI_F16, 64>(t, map, stream) : launch<SATORI_F16, 128>(t, map, stream);
    return a.head_dim <= 64 ? launch<SATORI_BF16, 64>(t, map, stream) : launch<SATORI_BF16, 128>(t, map, stream);
}

}  // namespace satori
