// What the operators around the paged KV cache share: the cache and the batch as kernels see them, the search for the
// sequence a token belongs to, and the 8-bit rows.
//
// Cache layout: K and V are [pages][kv_heads][page_size][head_dim], so that one head's page is one contiguous block. With
// 8 bits a row (one head of one token) holds e4m3 codes and one exponent e, value = code * 2^e; the exponents are
// [pages][kv_heads][page_size]. A power of two as the scale costs no precision (e4m3 is itself a floating-point format), makes
// the code of a value unambiguous (x * 2^-e is exact, so there is one rounding), and makes the value exact in bf16 and fp16.
#pragma once

#include "common.cuh"

namespace magb200 {

// Bits of the device word a kernel raises when it meets a table or a length that does not fit; nothing is read or written through it.
constexpr int kBatchWord = 2;                // word of the status buffer
constexpr int kWorkWord = 16;                // two words: work handed out by the running many-row kernel, its CTAs that have ended
constexpr int kBadPage = 1, kBadRows = 2, kBadLength = 4;
constexpr int kNanExponent = -128;           // a row that held an infinity or a NaN: it reads back as NaN
constexpr int kMinExponent = -126, kMaxExponent = 120;

struct KvCache {
    uint8_t *k, *v;
    int8_t *k_exp, *v_exp;                   // 8-bit cache only
    int64_t pages;
    int dtype, bits, page_size, page_shift, kv_heads, dim;
};
struct KvBatch {
    const int32_t *cu_q, *kv_len, *table;
    int32_t *status;
    int batch, max_pages;
    int64_t tokens;                          // rows of the packed q / k / v of the call
    int64_t max_q, max_kv;                   // the caller's bounds
};
struct RopeArgs {
    const int32_t *positions;
    const float *inv_freq;
    int rotary, interleaved;
    float factor;
};
// Rows of [tokens][heads][dim] with unit inner stride; strides in elements.
struct HeadRows {
    void *p;
    int64_t token_stride, head_stride;
    int heads;
};

// `early` in the launchers: launch as a programmatic dependent, so that the launch and the set-up run beside the tail of the kernel
// before it. Every kernel here begins with wait_for_predecessor() in all its threads.
int launch_qk_norm_rope(int dtype, int64_t tokens, int dim, const HeadRows &q, const HeadRows &k, const void *q_weight, const void *k_weight,
                        float eps, const RopeArgs &rope, const HeadRows &q_out, const HeadRows &k_out, cudaStream_t st, bool early);
int launch_kv_write(const KvCache &c, const KvBatch &b, const HeadRows &k, const HeadRows &v, cudaStream_t st, bool early);
int launch_kv_read(const KvCache &c, const KvBatch &b, const int32_t *cu_kv, const HeadRows &k, const HeadRows &v, cudaStream_t st, bool early);

struct AttentionArgs {
    KvCache cache;
    KvBatch batch;
    HeadRows q, out;
    float *lse;                              // [tokens][heads] or null
    int group;                               // query heads per KV head
    float scale_log2;                        // scale * log2(e)
    int causal;
    int64_t window;                          // 0: none
    int ctas;                                // multiprocessors that the tensor-core kernel may take
    float *partial;                          // workspace of split sequences
    size_t partial_bytes;
    int *arrived;                            // kMaxFewCtas words, zero between launches: parts done of the pair that begins in a CTA
};
constexpr int kMaxFewCtas = 1 << 12;
size_t attention_workspace_bytes();      // parts; the words of `arrived` lie behind them
int launch_paged_attention(const AttentionArgs &a, cudaStream_t st, bool early);
// How the rows of a call are dealt out, decided on the host from the caller's bounds. Sequences of at most `few_rows` (token,
// query head) rows go to the streaming kernel in tiles of few_tile rows, on few_ctas CTAs with pieces of at least few_least groups
// of 16 cached rows; all others to the tensor-core kernel in tiles of 256. 0 CTAs, 0 tiles: the kernel is not launched.
struct AttentionPlan {
    int few_rows;
    int few_tile, few_ctas, few_least;
    int64_t many_tiles, many_keys;   // upper bounds: the 256-row tiles of all sequences, the cached rows that a tile sees
};
AttentionPlan plan_attention(const KvCache &c, const KvBatch &b, int heads, bool causal, int64_t window, int sms);
int launch_attend_many(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early);
int launch_join_many(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st);     // if units may have been cut

#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_predecessor() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// The next kernel on the stream, if it is a programmatic dependent, may begin once every CTA has come by here (or ended).
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... Params, typename... Args>
inline int launch_kernel(void (*kernel)(Params...), dim3 grid, int threads, int shared, cudaStream_t st, bool early, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)shared;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 1 : 0;
    MAGB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
    count_launch();
    return MAGB200_OK;
}

// Largest b in [0, n) with cu[b] <= t, by a whole warp: 32 probes a step, so 1024 sequences cost two loads. cu ascends from 0.
__device__ __forceinline__ int find_sequence(const int32_t *__restrict__ cu, int n, int64_t t, int lane) {
    int lo = 0, left = n;
    while (left > 1) {
        const int step = (left + 31) >> 5;
        const int at = lo + lane * step;
        const bool below = at < lo + left && (int64_t)cu[at] <= t;
        const int hit = __popc(__ballot_sync(0xFFFFFFFFu, below));
        if (hit == 0) return lo;
        const int end = lo + left;
        lo += (hit - 1) * step;
        left = end - lo < step ? end - lo : step;
    }
    return lo;
}

// Row exponent: the least e with amax <= 448 * 2^e. `top`: bits of amax (a float without its sign).
__device__ __forceinline__ int row_exponent(uint32_t top) {
    if (top >= 0x7F800000u) return kNanExponent;
    // top = 1.m * 2^x with x = exponent field - 127; 448 = 1.75 * 2^8. Subnormal floats come out below the least exponent.
    const int x = (int)(top >> 23) - 127;
    const int e = x - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < kMinExponent ? kMinExponent : e;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// Codes of two numbers scaled by 2^-e: saturating round to nearest even, element 0 in the low byte. Beyond 240 the next code may
// stand for a number past the largest finite one of the tensor's type (fp16 at e = 8, bf16 at e = 120): there `most` is 240.
__device__ __forceinline__ uint32_t pack2_e4m3(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
template <int DT> __device__ __forceinline__ float most_code(int e) { return e >= (DT == MAGB200_F16 ? 8 : kMaxExponent) ? 240.0f : 448.0f; }

// Two codes -> two floats (exact), element 0 from the low byte.
__device__ __forceinline__ float2 unpack2_e4m3(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    float2 f;
    unpack2<MAGB200_F16>(h, f.x, f.y);
    return f;
}
// 2^e for reading a row; the exponent of a non-finite row gives NaN.
__device__ __forceinline__ float row_scale(int e) { return e == kNanExponent ? __uint_as_float(0x7FC00000u) : pow2f(e); }
#endif

}  // namespace magb200
