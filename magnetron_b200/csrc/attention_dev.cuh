// Device code that both attention kernels use: the rows and the cached rows of a tile, splits, asynchronous copies, codes.
#pragma once

#include "attention.cuh"

#include <atomic>
#include <math_constants.h>

namespace magb200 {
namespace {

constexpr float kLn2 = 0.6931471805599453f;

// ---- a tile of rows of one sequence ---------------------------------------------------------------------------------------
// Positions, rows and lengths fit 32 bits (the host refuses more); offsets into memory are 64 bits.
struct Tile {
    int q_begin;              // first row of the packed q of this sequence
    int q_len, kv_len, rows;
    int lo, hi;               // cached rows that any row of the tile may see; lo is on a 16-row boundary
};
// Lengths are read from device memory, so they are checked here: what does not fit raises the word and is cut off.
__device__ __forceinline__ bool sequence_of(const AttentionArgs &a, int b, Tile &t) {
    const int begin = a.batch.cu_q[b], end = a.batch.cu_q[b + 1];
    int kv = a.batch.kv_len[b];
    const int64_t table = (int64_t)a.batch.max_pages * a.cache.page_size;
    const int room = table > 0x7FFFF000 ? 0x7FFFF000 : (int)table;       // positions fit 32 bits with room for a block
    if (begin < 0 || end < begin || end > a.batch.tokens || end - begin > a.batch.max_q) { atomicOr(a.batch.status + kBatchWord, kBadRows); return false; }
    if (kv > room) { atomicOr(a.batch.status + kBatchWord, kBadLength); kv = room; }
    if (kv < 0) {
        if (end > begin) atomicOr(a.batch.status + kBatchWord, kBadLength);
        kv = 0;
    }
    t.q_begin = begin;
    t.q_len = end - begin;
    t.kv_len = kv;
    t.rows = t.q_len * a.group;
    return t.q_len > 0;
}
__device__ __forceinline__ void span_of(const AttentionArgs &a, int row0, int tile_rows, Tile &t) {
    t.lo = 0;
    t.hi = t.kv_len;
    if (a.causal) {
        const int last = (t.rows - row0 > tile_rows ? row0 + tile_rows : t.rows) - 1;
        const int shift = t.kv_len - t.q_len;                           // position of new token i is shift + i
        const int top = shift + last / a.group + 1;
        t.hi = top < t.kv_len ? (top > 0 ? top : 0) : t.kv_len;
        const int64_t from = (int64_t)shift + row0 / a.group + 1 - a.window;
        if (a.window > 0 && from > 0) t.lo = (int)from & ~15;
    }
    if (t.lo > t.hi) t.lo = t.hi & ~15;
}
// Opts `kernel` in to `bytes` of shared memory on the current device, once per device.
template <auto *kernel, int bytes> inline int opt_in_shared() {
    static std::atomic<uint64_t> done{0};                               // of this kernel: one bit per device
    int device = 0;
    MAGB200_CUDA_TRY(cudaGetDevice(&device));
    if (device < 64 && (done.load(std::memory_order_relaxed) >> device & 1)) return MAGB200_OK;
    MAGB200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
    return MAGB200_OK;
}

// ---- PTX ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool valid) {   // not valid: sixteen zero bytes
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace
}  // namespace magb200
