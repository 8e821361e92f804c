// batch.cuh -- device view of a decode batch's plan, and the launch interfaces of its kernels.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged.h"

namespace satori {

// The plan as the kernels read it: this header, then the arrays it gives the offsets of (in ints from the
// header's start).  Everything that changes from step to step is behind the one pointer, the work buffers
// included, so captured launches read the current step's plan and write the buffers that it was sized for.
struct DevPlan {
    float *part_o;                   // partial records of record_rows x head_dim, not normalised
    float2 *part_ml;                 // [record][record_rows]: running maximum (log2 units) and sum
    const double *rope;              // [row][rotary / 2] (cos, sin)
    PlanHeader head;
    int row_position, row_page, row_slot, chain_off, chain, seg_rows, pages, cta_off, slots, items, merges;
};

template <typename T>
__device__ __forceinline__ const T *plan_array(const DevPlan *plan, int offset)
{
    return reinterpret_cast<const T *>(reinterpret_cast<const int *>(plan) + offset);
}

struct BatchAttn {
    const DevPlan *plan;
    const uint8_t *pool;             // the layer's pages
    int page_tokens, kv_heads, group, head_dim, type;
    const void *q;                   // rows of q_heads * head_dim elements of the cache's type, ldq apart
    long long ldq;
    void *out;                       // the same, of the cache's type or float
    long long ldo;
    int out_f32;
    float scale_log2;                // log2(e) / sqrt(head_dim)
    int ctas;
    unsigned *err;
};

// Whether two tensors of `rows` rows have a byte in common: rows of wa bytes la apart from a on, of wb bytes lb apart
// from b on.  Rows of the same distance that lie side by side (slices of wider ones) have none; of other distances
// anything that is not one before the other counts.
inline bool rows_overlap(const void *a, long long la, long long wa, const void *b, long long lb, long long wb, long long rows)
{
    const long long x = (long long)(uintptr_t)a, y = (long long)(uintptr_t)b;
    if (x + (rows - 1) * la + wa <= y || y + (rows - 1) * lb + wb <= x) return false;
    if (la != lb) return true;
    const long long at = ((y - x) % la + la) % la;
    return !(at >= wa && at + wb <= la);
}

// The kernels' share of PlanShape: tile and block sizes, costs and the CTAs a GPU holds at once.
void wide_plan_shape(int sm_count, PlanShape &shape);
int wide_record_rows();
cudaError_t launch_wide_attention(const BatchAttn &a, cudaStream_t stream);

// The tensor-core kernel of 16-bit caches with heads of up to 128.
bool tensor_attention_takes(int type, int head_dim);
void tensor_plan_shape(int sm_count, PlanShape &shape);
int tensor_record_rows();
// The cache as a tensor of (layer, page, K or V, head) blocks.
cudaError_t make_page_map(CUtensorMap *map, void *memory, int type, int head_dim, int page_tokens, unsigned long long blocks);
cudaError_t launch_tensor_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream);

// The kernel of FP32 caches with heads of up to 128.
bool f32_attention_takes(int type, int head_dim);
void f32_plan_shape(int head_dim, int sm_count, PlanShape &shape);
int f32_record_rows();
cudaError_t launch_f32_attention(const BatchAttn &a, const CUtensorMap &map, int layer_block, cudaStream_t stream);

// Merges the partial records of every row that has more than one source and writes its outputs.
// A record holds record_rows rows; by_column: as [head_dim / 4][row] groups of 4 values, otherwise [row][head_dim].
// `merges` (the plan's) chooses the launch's shape; any number is worked through.
cudaError_t launch_combine(const BatchAttn &a, int record_rows, int tile_m, bool by_column, int merges, int sm_count,
                           cudaStream_t stream);

// A launch that may start while the kernel before it on the stream still runs; it waits for that kernel's
// results itself (pdl_wait).
template <typename K, typename... Args>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// --------------------------------------------------------------------------- element types
template <int TYPE>
struct Elem;
template <>
struct Elem<SATORI_F32> {
    typedef float type;
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
    static __device__ __forceinline__ float from_double(double v) { return (float)v; }
};
template <>
struct Elem<SATORI_F16> {
    typedef __half type;
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ __half from_double(double v) { return __double2half(v); }
};
template <>
struct Elem<SATORI_BF16> {
    typedef __nv_bfloat16 type;
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_double(double v) { return __double2bfloat16(v); }
};

}  // namespace satori
