// pages.cu -- the paged key/value cache: its C ABI and the kernel that copies pages.
//
// The reference keeps one contiguous cache per session (src/Satori.Core/Model/DenseSession.cs:80-84) and can
// only reset it; a host that serves many requests needs to share a prompt's cache between them, to branch a
// request and to give memory back.  Here a cache is an array of pages of `page_tokens` tokens; a sequence is
// a list of page numbers, and forking one shares its full pages.
//
// Page copies (a fork's or rewind's partly filled page, a compaction's moves) are one launch for all pairs
// and all layers.  A copy reads and writes every byte once, so HBM bounds it.
#include "batch.cuh"
#include "common.cuh"
#include "paged_internal.h"

#include <string.h>

#include <algorithm>
#include <unordered_map>

using namespace satori;

namespace {

// Page pairs travel as a kernel parameter (at most 32,764 bytes), so a copy needs no upload that a later
// call could overwrite.  Three sizes: the launch's cost on the host grows with the parameter.
constexpr int kFewPairs = 56, kSomePairs = 480, kManyPairs = 4000;
template <int N>
struct PagePairs {
    int from[N], to[N];
};

constexpr int kCopyThreads = 256, kCopyUnroll = 4;     // 16-byte words: one block copies 16 KB

// Block (x, y, z): 16 KB piece x of pair y in layer z (y and z stride over what the grid does not cover).
// No pair's destination is another pair's source or destination.
template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(uint8_t *memory, size_t layer_bytes,
                                                                  size_t block_bytes, int layers, int pairs,
                                                                  const __grid_constant__ PagePairs<N> list)
{
    const size_t words = block_bytes / 16;
    const size_t i0 = (size_t)blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
    for (int layer = blockIdx.z; layer < layers; layer += gridDim.z)
        for (int p = blockIdx.y; p < pairs; p += gridDim.y) {
            uint8_t *base = memory + (size_t)layer * layer_bytes;
            const uint4 *src = reinterpret_cast<const uint4 *>(base + (size_t)list.from[p] * block_bytes);
            uint4 *dst = reinterpret_cast<uint4 *>(base + (size_t)list.to[p] * block_bytes);
            uint4 v[kCopyUnroll];
#pragma unroll
            for (int u = 0; u < kCopyUnroll; ++u)
                if (i0 + u * kCopyThreads < words) v[u] = __ldcs(src + i0 + u * kCopyThreads);
#pragma unroll
            for (int u = 0; u < kCopyUnroll; ++u)
                if (i0 + u * kCopyThreads < words) __stcs(dst + i0 + u * kCopyThreads, v[u]);
        }
}

template <int N>
cudaError_t launch_copy(const satori_pages *p, const int *pairs, int n, cudaStream_t stream)
{
    PagePairs<N> list;
    for (int i = 0; i < n; ++i) {
        list.from[i] = pairs[2 * i];
        list.to[i] = pairs[2 * i + 1];
    }
    const size_t bytes = p->block_bytes(), piece = (size_t)kCopyThreads * kCopyUnroll * 16;
    const dim3 grid((unsigned)((bytes + piece - 1) / piece), (unsigned)n, (unsigned)std::min(p->layers, 65535));
    copy_pages_kernel<N><<<grid, kCopyThreads, 0, stream>>>(p->memory, p->layer_bytes(), bytes, p->layers, n, list);
    return cudaGetLastError();
}

// Queues the copies of p->copies on the context's stream.
int copy_pages(satori_pages *p)
{
    if (!p->ctx || p->copies.empty()) return SATORI_OK;
    DeviceScope scope(p->ctx->device);
    if (scope.status != cudaSuccess) return cuda_fail(scope.status, "cudaSetDevice");
    const int n = (int)(p->copies.size() / 2);
    for (int i = 0; i < n; i += kManyPairs) {
        const int some = std::min(n - i, kManyPairs);
        const int *pairs = p->copies.data() + 2 * (size_t)i;
        cudaStream_t stream = p->ctx->stream;
        cudaError_t e = some <= kFewPairs    ? launch_copy<kFewPairs>(p, pairs, some, stream)
                        : some <= kSomePairs ? launch_copy<kSomePairs>(p, pairs, some, stream)
                                             : launch_copy<kManyPairs>(p, pairs, some, stream);
        if (e != cudaSuccess) return cuda_fail(e, "copy pages");
    }
    return SATORI_OK;
}

int check_pages(satori_pages *p)
{
    if (!p || p->disposed) return set_error(SATORI_ERR_DISPOSED, "paged cache is disposed");
    return SATORI_OK;
}

// A replayed graph would repeat a copy but not the change of the tables that goes with it.
int check_not_capturing(const satori_pages *p)
{
    if (!p->ctx) return SATORI_OK;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(p->ctx->stream, &status);
    if (e != cudaSuccess) return cuda_fail(e, "cudaStreamIsCapturing");
    if (status != cudaStreamCaptureStatusNone)
        return set_error(SATORI_ERR_NOT_SUPPORTED, "page tables cannot change inside a stream capture");
    return SATORI_OK;
}

// The device answers, before a table changes for it.
int check_device(const satori_pages *p)
{
    if (!p->ctx) return SATORI_OK;
    DeviceScope scope(p->ctx->device);
    return scope.status == cudaSuccess ? SATORI_OK : cuda_fail(scope.status, "cudaSetDevice");
}

// Every id names a live sequence; with `distinct`, none comes twice.
int check_sequences(satori_pages *p, int n, const int *seqs, bool distinct)
{
    if (n < 0 || (n > 0 && !seqs)) return set_error(SATORI_ERR_ARGUMENT, "bad sequence list");
    for (int i = 0; i < n; ++i)
        if (!p->tables.find(seqs[i])) return set_error(SATORI_ERR_ARGUMENT, "sequence %d does not exist", seqs[i]);
    if (distinct && n > 1) {
        std::vector<int> sorted(seqs, seqs + n);
        std::sort(sorted.begin(), sorted.end());
        if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
            return set_error(SATORI_ERR_ARGUMENT, "a sequence is listed twice");
    }
    return SATORI_OK;
}

int check_room(satori_pages *p, long long need)
{
    if (need > p->tables.free_pages())
        return set_error(SATORI_ERR_CONTEXT_FULL, "the cache has %d free pages of %d; %lld are needed",
                         p->tables.free_pages(), p->tables.pages(), need);
    return SATORI_OK;
}

int pages_needed(int tokens, int page_tokens) { return (int)(((long long)tokens + page_tokens - 1) / page_tokens); }

// Whether rewinding the sequences frees more pages than its copies take.
bool makes_room(const satori_pages *p, int n, const int *seqs, const int *positions)
{
    PageTables &tables = const_cast<satori_pages *>(p)->tables;
    const int pt = tables.page_tokens();
    std::unordered_map<int, int> fewer;              // page -> references that the call takes away
    long long gain = 0;
    for (int i = 0; i < n; ++i) {
        const PageSequence &s = *tables.find(seqs[i]);
        for (size_t j = (size_t)pages_needed(positions[i], pt); j < s.pages.size(); ++j)
            gain += ++fewer[s.pages[j]] == tables.refs(s.pages[j]);
    }
    for (int i = 0; i < n; ++i) {
        if (positions[i] % pt == 0) continue;
        const int page = tables.find(seqs[i])->pages[positions[i] / pt];
        int &gone = fewer[page];
        if (tables.refs(page) - gone == 1) continue;
        ++gone;                                      // it leaves the page to the others, for a copy
        --gain;
    }
    return gain > 0;
}

}  // namespace

int satori::pages_extend(satori_pages *p, int n, const int *seqs, const int *counts)
{
    int rc = check_sequences(p, n, seqs, true);
    if (rc) return rc;
    if (n > 0 && !counts) return set_error(SATORI_ERR_ARGUMENT, "counts is null");
    long long need = 0;
    for (int i = 0; i < n; ++i) {
        const PageSequence &s = *p->tables.find(seqs[i]);
        if (counts[i] < 0) return set_error(SATORI_ERR_ARGUMENT, "count %d is negative", counts[i]);
        if (counts[i] > 0x7fffffff - s.length) return set_error(SATORI_ERR_ARGUMENT, "sequence length exceeds Int32 limits");
        need += pages_needed(s.length + counts[i], p->tables.page_tokens()) - (long long)s.pages.size();
    }
    if ((rc = check_room(p, need))) return rc;
    for (int i = 0; i < n; ++i) {                    // what can fail comes before the first change
        PageSequence &s = *p->tables.find(seqs[i]);
        const size_t pages = (size_t)pages_needed(s.length + counts[i], p->tables.page_tokens());
        if (pages > s.pages.capacity()) s.pages.reserve(std::max(pages, 2 * s.pages.capacity()));
    }
    for (int i = 0; i < n; ++i) {
        PageSequence &s = *p->tables.find(seqs[i]);
        if (counts[i] == 0) continue;
        s.length += counts[i];
        const size_t pages = (size_t)pages_needed(s.length, p->tables.page_tokens());
        while (s.pages.size() < pages) s.pages.push_back(p->tables.take());
        ++s.version;
    }
    return SATORI_OK;
}

void satori::pages_shrink(satori_pages *p, int n, const int *seqs, const int *counts)
{
    for (int i = 0; i < n; ++i) {
        PageSequence &s = *p->tables.find(seqs[i]);
        s.length -= counts[i];
        const size_t keep = (size_t)pages_needed(s.length, p->tables.page_tokens());
        for (; s.pages.size() > keep; s.pages.pop_back()) p->tables.release(s.pages.back());
        ++s.version;
    }
}

static void free_pages_memory(satori_pages *p)
{
    if (p->owned && p->memory) {
        DeviceScope scope(p->ctx->device);
        cudaStreamSynchronize(p->ctx->stream);
        cudaFree(p->memory);
    }
    p->memory = nullptr;
}

void satori::pages_unref(satori_pages *p)
{
    if (--p->users == 0 && p->disposed) delete p;
}

extern "C" int satori_pages_create(satori_ctx *ctx, int layers, int pages, int page_tokens, int kv_heads, int head_dim,
                                   int type, void *memory, satori_pages **out)
{
    return guarded([&]() -> int {
        if (!out) return set_error(SATORI_ERR_ARGUMENT, "out is null");
        if (layers <= 0 || pages <= 0 || kv_heads <= 0)
            return set_error(SATORI_ERR_ARGUMENT, "layers/pages/kv_heads must be positive");
        if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)))
            return set_error(SATORI_ERR_ARGUMENT, "page_tokens must be 16, 32, 64, 128 or 256");
        if (head_dim <= 0) return set_error(SATORI_ERR_ARGUMENT, "head_dim must be positive");
        if (head_dim > 256 || head_dim % 8)
            return set_error(SATORI_ERR_NOT_SUPPORTED, "head_dim must be a multiple of 8, at most 256");
        if (!type_size(type)) return set_error(SATORI_ERR_ARGUMENT, "unsupported type %d", type);
        // Blocks of (layer, page, K or V, head) are numbered in 32 bits.
        if ((double)layers * pages * 2 * kv_heads > 2147483647.0)
            return set_error(SATORI_ERR_NOT_SUPPORTED, "layers * pages * 2 * kv_heads exceeds Int32 limits");
        if (memory && !ctx) return set_error(SATORI_ERR_ARGUMENT, "memory without a context");
        if ((uintptr_t)memory % 16) return set_error(SATORI_ERR_ARGUMENT, "memory must be 16-byte aligned");
        satori_pages *p = new satori_pages(pages, page_tokens);
        p->ctx = ctx;
        p->layers = layers;
        p->kv_heads = kv_heads;
        p->head_dim = head_dim;
        p->type = type;
        p->memory = (uint8_t *)memory;
        if (ctx && !memory) {
            DeviceScope scope(ctx->device);
            cudaError_t e = scope.status;
            if (e == cudaSuccess) e = cudaMalloc(&p->memory, p->layer_bytes() * (size_t)layers);
            if (e != cudaSuccess) {
                delete p;
                return cuda_fail(e, "allocate paged cache");
            }
            p->owned = true;
        }
        if (ctx && (tensor_attention_takes(type, head_dim) || f32_attention_takes(type, head_dim))) {
            DeviceScope scope(ctx->device);
            cudaError_t e = make_page_map(&p->map, p->memory, type, head_dim, page_tokens,
                                          (unsigned long long)layers * pages * 2 * kv_heads);
            if (e != cudaSuccess) {
                satori_pages_destroy(p);
                return cuda_fail(e, "describe the cache for TMA");
            }
        }
        *out = p;
        return SATORI_OK;
    });
}

extern "C" int satori_pages_info(const satori_pages *p, int *used, int *free_count, int *top, size_t *bytes, void **memory)
{
    int rc = check_pages(const_cast<satori_pages *>(p));
    if (rc) return rc;
    if (used) *used = p->tables.pages() - p->tables.free_pages();
    if (free_count) *free_count = p->tables.free_pages();
    if (top) *top = p->tables.top();
    if (bytes) *bytes = p->layer_bytes() * (size_t)p->layers;
    if (memory) *memory = p->memory;
    return SATORI_OK;
}

extern "C" int satori_pages_new(satori_pages *p, int n, int *seqs)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        if (rc) return rc;
        if (n < 0 || (n > 0 && !seqs)) return set_error(SATORI_ERR_ARGUMENT, "bad sequence list");
        if (!p->tables.room_for_sequences(n)) return set_error(SATORI_ERR_CONTEXT_FULL, "too many sequences");
        std::vector<int> ids;
        ids.reserve((size_t)n);
        try {
            for (int i = 0; i < n; ++i) ids.push_back(p->tables.add());
        } catch (...) {
            for (int id : ids) p->tables.remove(id);
            throw;
        }
        std::copy(ids.begin(), ids.end(), seqs);
        return SATORI_OK;
    });
}

extern "C" int satori_pages_extend(satori_pages *p, int n, const int *seqs, const int *counts)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        return rc ? rc : pages_extend(p, n, seqs, counts);
    });
}

extern "C" int satori_pages_fork(satori_pages *p, int n, const int *parents, const int *positions, int share,
                                 int *children)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        if (rc) return rc;
        if ((rc = check_sequences(p, n, parents, false)) || (rc = check_not_capturing(p))) return rc;
        if (n > 0 && !children) return set_error(SATORI_ERR_ARGUMENT, "children is null");
        if (!p->tables.room_for_sequences(n)) return set_error(SATORI_ERR_CONTEXT_FULL, "too many sequences");
        const int pt = p->tables.page_tokens();
        long long need = 0;
        for (int i = 0; i < n; ++i) {
            const PageSequence &s = *p->tables.find(parents[i]);
            const int at = positions ? positions[i] : s.length;
            if (at < 0 || at > s.length)
                return set_error(SATORI_ERR_ARGUMENT, "position %d is outside sequence %d (%d tokens)", at, parents[i], s.length);
            need += pages_needed(at, pt) - (share ? at / pt : 0);
        }
        if ((rc = check_room(p, need)) || (rc = check_device(p))) return rc;
        std::vector<int> copies, ids;
        copies.reserve(2 * (size_t)need);
        ids.reserve((size_t)n);
        try {
            for (int i = 0; i < n; ++i) {
                ids.push_back(p->tables.add());
                p->tables.find(ids.back())->pages.reserve(
                    (size_t)pages_needed(positions ? positions[i] : p->tables.find(parents[i])->length, pt));
            }
        } catch (...) {
            for (int id : ids) p->tables.remove(id);
            throw;
        }
        for (int i = 0; i < n; ++i) {
            const PageSequence &s = *p->tables.find(parents[i]);
            PageSequence &child = *p->tables.find(ids[i]);
            child.length = positions ? positions[i] : s.length;
            const int whole = share ? child.length / pt : 0;
            for (int j = 0; j < pages_needed(child.length, pt); ++j) {
                if (j < whole) {
                    p->tables.share(s.pages[j]);
                    child.pages.push_back(s.pages[j]);
                } else {
                    child.pages.push_back(p->tables.take());
                    copies.push_back(s.pages[j]);
                    copies.push_back(child.pages.back());
                }
            }
        }
        p->copies.swap(copies);
        if ((rc = copy_pages(p))) {
            for (int id : ids) p->tables.remove(id);
            return rc;
        }
        std::copy(ids.begin(), ids.end(), children);
        return SATORI_OK;
    });
}

extern "C" int satori_pages_rewind(satori_pages *p, int n, const int *seqs, const int *positions)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        if (rc) return rc;
        if ((rc = check_sequences(p, n, seqs, true)) || (rc = check_not_capturing(p))) return rc;
        if (n > 0 && !positions) return set_error(SATORI_ERR_ARGUMENT, "positions is null");
        const int pt = p->tables.page_tokens();
        long long split = 0;                         // sequences that end inside a page: it may be shared
        for (int i = 0; i < n; ++i) {
            const PageSequence &s = *p->tables.find(seqs[i]);
            if (positions[i] < 0 || positions[i] > s.length)
                return set_error(SATORI_ERR_ARGUMENT, "position %d is outside sequence %d (%d tokens)", positions[i],
                                 seqs[i], s.length);
            const int whole = positions[i] / pt;
            split += positions[i] % pt && p->tables.refs(s.pages[whole]) > 1;
        }
        // The pages that this call frees may serve it, and a page may be shared no more when its turn comes: with
        // too few free pages for the least favourable order, the counts are tried on a copy.
        if (split > p->tables.free_pages() && !makes_room(p, n, seqs, positions)) return check_room(p, split);
        if ((rc = check_device(p))) return rc;
        std::vector<int> copies;
        copies.reserve(2 * (size_t)split);
        for (int i = 0; i < n; ++i) {
            PageSequence &s = *p->tables.find(seqs[i]);
            const size_t keep = (size_t)pages_needed(positions[i], pt);
            if (positions[i] == s.length) continue;
            for (size_t j = keep; j < s.pages.size(); ++j) p->tables.release(s.pages[j]);
            s.pages.resize(keep);
            s.length = positions[i];
            ++s.version;
        }
        // All releases come first: a page that is copied from here has another owner, so it is neither free
        // nor a destination.
        for (int i = 0; i < n; ++i) {
            PageSequence &s = *p->tables.find(seqs[i]);
            if (s.length % pt == 0 || p->tables.refs(s.pages.back()) == 1) continue;
            const int page = s.pages.back();
            s.pages.back() = p->tables.take();
            p->tables.release(page);
            copies.push_back(page);
            copies.push_back(s.pages.back());
        }
        p->copies.swap(copies);
        return copy_pages(p);
    });
}

extern "C" int satori_pages_free(satori_pages *p, int n, const int *seqs)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        if (rc) return rc;
        if ((rc = check_sequences(p, n, seqs, true))) return rc;
        for (int i = 0; i < n; ++i) p->tables.remove(seqs[i]);
        return SATORI_OK;
    });
}

extern "C" int satori_pages_compact(satori_pages *p, int *moved)
{
    return guarded([&]() -> int {
        int rc = check_pages(p);
        if (rc) return rc;
        if ((rc = check_not_capturing(p)) || (rc = check_device(p))) return rc;
        p->tables.compact(p->copies);
        if (moved) *moved = (int)(p->copies.size() / 2);
        return copy_pages(p);
    });
}

extern "C" int satori_pages_table(satori_pages *p, int seq, int *length, int *pages, int capacity, int *count)
{
    int rc = check_pages(p);
    if (rc) return rc;
    if ((rc = check_sequences(p, 1, &seq, false))) return rc;
    const PageSequence &s = *p->tables.find(seq);
    if (capacity < 0 || (capacity > 0 && !pages)) return set_error(SATORI_ERR_ARGUMENT, "bad page list");
    if (length) *length = s.length;
    if (count) *count = (int)s.pages.size();
    std::copy_n(s.pages.begin(), std::min((size_t)capacity, s.pages.size()), pages);
    return SATORI_OK;
}

extern "C" int satori_pages_copies(satori_pages *p, int *pairs, int capacity, int *count)
{
    int rc = check_pages(p);
    if (rc) return rc;
    if (capacity < 0 || (capacity > 0 && !pairs)) return set_error(SATORI_ERR_ARGUMENT, "bad pair list");
    if (count) *count = (int)(p->copies.size() / 2);
    std::copy_n(p->copies.begin(), std::min(2 * (size_t)capacity, p->copies.size()), pairs);
    return SATORI_OK;
}

extern "C" int satori_pages_destroy(satori_pages *p)
{
    if (!p || p->disposed) return SATORI_OK;
    free_pages_memory(p);
    p->disposed = true;
    if (p->users == 0) delete p;
    return SATORI_OK;
}
