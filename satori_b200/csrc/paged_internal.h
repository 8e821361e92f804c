// paged_internal.h -- handles of the paged cache and of a decode batch.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <exception>
#include <new>
#include <vector>

#include "capi_internal.h"
#include "paged.h"

struct satori_pages {
    satori_ctx *ctx = nullptr;                 // null: the tables only
    int layers = 0, kv_heads = 0, head_dim = 0, type = 0;
    satori::PageTables tables;
    uint8_t *memory = nullptr;                 // [layer][page][K, V][kv_head][token][dim]
    bool owned = false;                        // allocated here
    bool disposed = false;
    int users = 0;                             // decode batches that point here
    alignas(64) CUtensorMap map = {};          // the memory as the tensor-core attention loads it
    std::vector<int> copies;                   // (from, to) page pairs of the last fork / rewind / compact

    satori_pages(int pages, int page_tokens) : tables(pages, page_tokens) {}
    size_t block_bytes() const                 // one page of one layer, K and V
    {
        return (size_t)2 * kv_heads * tables.page_tokens() * head_dim * satori::type_size(type);
    }
    size_t layer_bytes() const { return block_bytes() * (size_t)tables.pages(); }
};

namespace satori {

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(F f)
{
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return set_error(SATORI_ERR_OUT_OF_MEMORY, "out of host memory");
    } catch (const std::exception &e) {
        return set_error(SATORI_ERR_ARGUMENT, "%s", e.what());
    }
}

// Adds `counts[i]` tokens to each sequence or changes nothing (satori_pages_extend without its null checks).
int pages_extend(satori_pages *p, int n, const int *seqs, const int *counts);
void pages_shrink(satori_pages *p, int n, const int *seqs, const int *counts);     // takes pages_extend back
void pages_unref(satori_pages *p);             // a batch lets go of its cache

}  // namespace satori
