// Attention of new tokens over the paged KV cache.
//
//   out = softmax(scale * q K^T + mask) V      per sequence and head, rows that the mask leaves empty give 0 and lse = -inf
//
// The query heads that share a KV head are rows of the same tiles: row r of a sequence is (new token r / group, query head
// r % group), so that a cached row is read once for the whole group. One pass over the cached rows with the running maximum
// and sum of the softmax (exp2 of scores scaled by log2 e), both in fp32, as are the output's sums; the weights are rounded
// to 16 bits for their product with V: to the tensor type, or to fp16 for few rows over codes. Long sequences are split along the cached rows over several CTAs, which leave
// (maximum, sum, output) of their part in the workspace, to be joined in the order of the parts.
#include "attention_dev.cuh"

#include <math.h>

namespace magb200 {
namespace {

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == MAGB200_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- few rows: stream the cache past 8 or 16 rows -----------------------------------------------------------------------------
// Bound by HBM: a row tile of 8 (token, head) rows needs 16 flop per cached byte. Each warp walks its own tiles of cached rows
// through a private ring in shared memory (16-byte asynchronous copies), multiplies with mma.sync m16n8k16 and keeps its own
// maximum, sum and output; the warps meet once at the end. The cached rows are the 16 of the instruction and the queries its
// 8 columns: S^T = K Q^T and O^T = V^T P^T, so that the eight rows or fewer of a decode step fill the instruction (as its 16 rows
// they left half of it and half of the softmax empty; tcgen05 would need 128). P^T comes from S^T by a transposition of 8 x 8
// matrices between the lanes (movmatrix). 8-bit rows stay codes in shared memory and become fp16 numbers in the registers (one
// conversion per two codes); their exponents go to the scores and to the weights, never to the elements.
constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps;
template <bool kEight, int NT> struct FewCfg {                     // NT: groups of 8 rows
    // CTAs on a multiprocessor; us of 64 sequences on up to 4096 rows, 8 KV heads of 128, with two and with three: 16 bits and 8 rows 130
    // and 136, 16 rows 140 and 149; 8 bits and 8 rows 106 and 89 (four: 124), 16 rows 136 and 182
    static constexpr int kPerSm = NT == 1 && kEight ? 3 : 2;
    static constexpr int kStages = 2;
    // groups of 16 cached rows in a tile: with codes two groups give a warp twice the independent work between two waits
    static constexpr int kSubs = kEight ? 2 : 1;
    static constexpr int kTok = 16 * kSubs;
    static constexpr int pitch(int dpad) { return (kEight ? dpad : 2 * dpad) + 16; }   // 16 bytes off a multiple of 128: no bank conflicts
    static constexpr int stage_bytes(int dpad) { return 2 * kTok * pitch(dpad) + (kEight ? 2 * kTok : 0); }
    static constexpr int ring_bytes(int dpad) { return kFewWarps * kStages * stage_bytes(dpad); }
    static constexpr int merge_bytes(int dpad) { return kFewWarps * 8 * NT * (dpad + 8) * 4; }
    static constexpr int smem_bytes(int dpad) { return ring_bytes(dpad) > merge_bytes(dpad) ? ring_bytes(dpad) : merge_bytes(dpad); }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {      // an 8 x 8 matrix of 16-bit elements across the warp
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
// Two e4m3 codes of the low or the high half of a word as two fp16 numbers: exact.
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
    uint32_t d;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(w));
    return d;
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
    uint32_t d;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(w));
    return d;
}

// Cached rows of sequence b that the kernel walks, in groups of 16; 0: not a sequence of this kernel. One at least otherwise, for
// the rows of zeros of a sequence without cached rows. All its rows are one tile, so its last one sees the last cached row.
__device__ __forceinline__ int groups_of(const AttentionArgs &a, int b, int few_rows, Tile &t) {
    if (!sequence_of(a, b, t) || t.rows > few_rows) return 0;
    t.hi = t.kv_len;
    const int64_t from = (int64_t)t.kv_len - t.q_len + 1 - a.window;
    t.lo = a.causal && a.window > 0 && from > 0 ? (int)from & ~15 : 0;
    if (t.lo > t.hi) t.lo = t.hi & ~15;
    return t.hi > t.lo ? (t.hi - t.lo + 15) >> 4 : 1;
}

// All (sequence, KV head) pairs' cached rows stand in one line, cut into equal pieces, one per CTA: a piece may end inside a pair
// and go on with the next, so that lengths that differ leave no multiprocessor idle (one part per CTA and a part per grid cell,
// chosen from the longest sequence, ran the long 8-bit decode as 1.05 waves: 114 us). A pair that lies in several pieces is
// joined by the last of their CTAs to finish. `least`: groups of 16 rows in a piece at least.
template <int DT, bool kEight, int DPAD, int NT>
__device__ __forceinline__ void attend_few(const AttentionArgs &a, int few_rows, int least) {
    using Cfg = FewCfg<kEight, NT>;
    constexpr int MM = kEight ? (int)MAGB200_F16 : DT;             // type of the products
    // fp16 weights are made 2^15 times as large, as far as the type reaches: they keep all their bits down to 2^-29 of the row's
    // largest and are lost under 2^-40 of it, where many rows of small weight would otherwise go missing from the output (under
    // 2^-25 unscaled: 0.2 % of 50000 rows) while the sum in fp32 counts them
    constexpr float kLift = MM == MAGB200_F16 ? 15.0f : 0.0f;
    constexpr int kSteps = DPAD / 16, kPitch = Cfg::pitch(DPAD), kStage = Cfg::stage_bytes(DPAD), kRows = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int is_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, c4 = lane & 3;
    const int dim = a.cache.dim, kv_heads = a.cache.kv_heads;

    // ---- where this CTA's piece begins: sequence b, KV head, groups `skip` of its `n`
    int b = 0, head = 0, n = 0;
    int quota, at, until, pair;                                     // `pair`: where the pair begins in the line
    Tile t;
    {
        // sequences 0 .. 31 are read once, by the lanes; more than those are counted first and searched afterwards
        int mine = lane < a.batch.batch ? groups_of(a, lane, few_rows, t) : 0;
        unsigned upto = (unsigned)mine;                             // below 2^32: 32 sequences of fewer than 2^27 groups
        auto scan = [&]() {
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const unsigned o = __shfl_up_sync(0xFFFFFFFFu, upto, s);
                if (lane >= s) upto += o;
            }
        };
        scan();
        int64_t sum = __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (a.batch.batch > 32) {
            int64_t rest = 0;
            for (int i = lane + 32; i < a.batch.batch; i += 32) { Tile x; rest += groups_of(a, i, few_rows, x); }
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) rest += __shfl_xor_sync(0xFFFFFFFFu, rest, x);
            sum += rest;
        }
        sum *= kv_heads;
        if (sum > 0x3FFFFFFF) {                                     // 2^34 cached rows of all heads: lengths that no memory holds
            atomicOr(a.batch.status + kBatchWord, kBadLength);
            return;
        }
        const int all = (int)sum;
        quota = (int)(((unsigned)all + gridDim.x - 1) / gridDim.x);
        if (quota < least) quota = least;
        if ((int64_t)quota * blockIdx.x >= all) return;
        at = quota * (int)blockIdx.x;
        until = all - at < quota ? all : at + quota;
        unsigned before = 0;                                        // from here on all sums are below 2^30
        for (int first = 0;;) {
            const uint32_t past = __ballot_sync(0xFFFFFFFFu, (int)(before + upto) * kv_heads > at);
            if (past) {
                const int hit = __ffs(past) - 1;
                b = first + hit;
                n = __shfl_sync(0xFFFFFFFFu, mine, hit);
                pair = (int)(before + __shfl_sync(0xFFFFFFFFu, upto, hit) - (unsigned)n) * kv_heads;
                t.q_begin = __shfl_sync(0xFFFFFFFFu, t.q_begin, hit);
                t.q_len = __shfl_sync(0xFFFFFFFFu, t.q_len, hit);
                t.kv_len = __shfl_sync(0xFFFFFFFFu, t.kv_len, hit);
                t.rows = __shfl_sync(0xFFFFFFFFu, t.rows, hit);
                t.lo = __shfl_sync(0xFFFFFFFFu, t.lo, hit);
                t.hi = __shfl_sync(0xFFFFFFFFu, t.hi, hit);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
            first += 32;
            if (first >= a.batch.batch) return;                     // not while the lengths stay as they were above
            mine = first + lane < a.batch.batch ? groups_of(a, first + lane, few_rows, t) : 0;
            upto = (unsigned)mine;
            scan();
        }
        head = (int)((unsigned)(at - pair) / (unsigned)n);
        pair += head * n;
    }
    // row / group for rows below 32, by a multiplication
    const unsigned by_group = 65536u / (unsigned)a.group + 1u;
    auto token_of = [&](int r) { return (int)(((unsigned)r * by_group) >> 16); };
    for (;;) {                                                      // pair after pair
        // this piece's part of the pair, and the CTAs that have the others
        const int begin = t.lo + (at > pair ? (at - pair) * 16 : 0);
        const int end = until - pair < n ? t.lo + (until - pair) * 16 : t.hi;
        const int first_cta = at > pair ? (int)((unsigned)pair / (unsigned)quota) : (int)blockIdx.x;
        const int used = end == t.hi && first_cta == (int)blockIdx.x ? 1 : (int)((unsigned)(pair + n - 1) / (unsigned)quota) - first_cta + 1;
        constexpr int kSubs = Cfg::kSubs, kTok = Cfg::kTok;
        const int tiles = end > begin ? (end - begin + kTok - 1) / kTok : 0;

        // ---- ring of this warp: [K rows][V rows][K exponents][V exponents] a stage
        uint8_t *ring = smem + warp * Cfg::kStages * kStage;
        const uint32_t ring_at = smem_addr(ring);
        const int32_t *table = a.batch.table + (int64_t)b * a.batch.max_pages;
        const int mine = tiles > warp ? (tiles - warp + kFewWarps - 1) / kFewWarps : 0;
        struct Pages { int of[kSubs]; };          // 16 cached rows lie in one page
        auto pages_of = [&](int i) {
            Pages p;
#pragma unroll
            for (int u = 0; u < kSubs; ++u) {
                const int row = begin + (warp + i * kFewWarps) * kTok + 16 * u;
                p.of[u] = i < mine && row < end ? table[row >> a.cache.page_shift] : 0;
            }
            return p;
        };
        constexpr int kChunks = (kEight ? DPAD : 2 * DPAD) / 16, kRowsPerCopy = 32 / kChunks;
        const int row_bytes = kEight ? dim : 2 * dim, copy_c = lane % kChunks, copy_r = lane / kChunks;
        const int from = copy_r * row_bytes + copy_c * 16, to = copy_r * kPitch + copy_c * 16;
        auto fetch = [&](int i, const Pages &pages) {
            if (i < mine) {
                const uint32_t dst = ring_at + (i % Cfg::kStages) * kStage;
#pragma unroll
                for (int u = 0; u < kSubs; ++u) {
                    const int row = begin + (warp + i * kFewWarps) * kTok + 16 * u;
                    const bool good = (uint32_t)pages.of[u] < (uint32_t)a.cache.pages;
                    if (!good && lane == 0) atomicOr(a.batch.status + kBatchWord, kBadPage);
                    // rows that are not wanted lie in the same page: their addresses are sound, and nothing is read from them
                    const int64_t cell = ((int64_t)(good ? pages.of[u] : 0) * a.cache.kv_heads + head) * a.cache.page_size + (row & (a.cache.page_size - 1));
                    const uint8_t *kp = a.cache.k + cell * row_bytes + from, *vp = a.cache.v + cell * row_bytes + from;
                    const int left = good ? end - row - copy_r : 0;
                    if (copy_c * 16 < row_bytes) {
#pragma unroll
                        for (int j = 0; j < 16; j += kRowsPerCopy) {
                            copy16(dst + (16 * u + j) * kPitch + to, kp + j * row_bytes, j < left);
                            copy16(dst + (kTok + 16 * u + j) * kPitch + to, vp + j * row_bytes, j < left);
                        }
                    }
                    if (kEight && lane < 2) copy16(dst + 2 * kTok * kPitch + kTok * lane + 16 * u, (lane ? a.cache.v_exp : a.cache.k_exp) + cell, good);
                }
            }
            copy_commit();
        };
        Pages next;
        {
            Pages p[Cfg::kStages];
#pragma unroll
            for (int i = 0; i < Cfg::kStages; ++i) p[i] = pages_of(i);
#pragma unroll
            for (int i = 0; i < Cfg::kStages - 1; ++i) fetch(i, p[i]);
            next = p[Cfg::kStages - 1];
        }

        // ---- the rows' queries, in the registers for the whole kernel. Against codes the product is in fp16, which holds every code;
        // bf16 queries are scaled by a power of two per row so that their largest element is in [1, 2), or in [2, 4) from 2^127 on, whose
        // reciprocal is below the least normal number: what falls below fp16's range then is under 2^-25 of it.
        uint32_t qf[NT][kSteps][2];               // columns g8 of each group of 8 rows
        float row_factor[NT][2];                  // of rows 2c and 2c + 1: scale * log2(e), and back from that power of two
        int last[NT][2], first[NT][2];            // cached rows first .. last - 1 are seen by these rows
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            const int r = m * 8 + g8;
            const bool live = r < t.rows;
            const int token = live ? token_of(r) : 0;
            const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q.p) + (int64_t)(t.q_begin + token) * a.q.token_stride +
                                  (int64_t)(head * a.group + (live ? r - token * a.group : 0)) * a.q.head_stride;
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t lo = 0, hi = 0;
                if (live && k * 16 < dim) {
                    // with codes the four neighbours 4c .. 4c + 3 of a step stand in the slots 2c, 2c + 1, 2c + 8, 2c + 9 of both operands
                    lo = *reinterpret_cast<const uint32_t *>(src + k * 16 + (kEight ? 4 * c4 : 2 * c4));
                    hi = *reinterpret_cast<const uint32_t *>(src + k * 16 + (kEight ? 4 * c4 + 2 : 2 * c4 + 8));
                }
                qf[m][k][0] = lo;
                qf[m][k][1] = hi;
                if constexpr (kEight && DT == MAGB200_BF16) top = max(top, max(max(lo & 0x7FFFu, (lo >> 16) & 0x7FFFu), max(hi & 0x7FFFu, (hi >> 16) & 0x7FFFu)));
            }
            float factor = a.scale_log2;
            if constexpr (kEight && DT == MAGB200_BF16) {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                int e = (int)(top >> 7) - 127;
                if (e < -126) e = -126;
                if (e == 127) e = 126;
                if (e == 128) e = 0;                                   // an infinity or a NaN stays one
                factor = a.scale_log2 * pow2f(e);
                const float inv = pow2f(-e);
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x, y;
                        unpack2<MAGB200_BF16>(qf[m][k][h], x, y);
                        qf[m][k][h] = pack2_rn<MAGB200_F16>(x * inv, y * inv);
                    }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                row_factor[m][j] = __shfl_sync(0xFFFFFFFFu, factor, 8 * c4 + 4 * j);
                const int row = m * 8 + 2 * c4 + j;
                const bool there = row < t.rows;
                const int pos = t.kv_len - t.q_len + (there ? token_of(row) : 0);
                last[m][j] = !there ? 0 : a.causal && pos + 1 < t.kv_len ? pos + 1 : t.kv_len;
                first[m][j] = a.window > 0 && (int64_t)pos + 1 - a.window > 0 ? (int)(pos + 1 - a.window) : 0;
            }
        }
        // every row of the tile sees all of the cached rows full_lo .. full_hi - 1
        int full_lo = 0, full_hi = t.kv_len;
        if (a.causal) {
            const int shift = t.kv_len - t.q_len;
            if (shift + 1 < full_hi) full_hi = shift + 1;
            const int64_t from = (int64_t)shift + t.q_len - a.window;
            if (a.window > 0 && from > 0) full_lo = (int)from;
        }

        // `top` is the running maximum of the scores, the reference of `sum` (with 16 bits 2^kLift times the sum of the weights). With codes
        // the output has a reference of its own, the maximum of score + exponent of the V row: the weights 2^(score + exponent - base)
        // are then at most 1 before the lift, however far the rows' exponents are apart.
        float acc[NT][kSteps][4];                 // elements (16 n + g8, + 8) or, with codes, (16 n + 2 g8, + 1) of rows 2c, 2c + 1
        float top[NT][2], base[NT][2], sum[NT][2];
#pragma unroll
        for (int m = 0; m < NT; ++m) {
#pragma unroll
            for (int n = 0; n < kSteps; ++n) { acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.0f; }
            top[m][0] = top[m][1] = base[m][0] = base[m][1] = -CUDART_INF_F;
            sum[m][0] = sum[m][1] = 0.0f;
        }

        for (int i = 0; i < mine; ++i) {
            copy_wait<Cfg::kStages - 2>();
            __syncwarp();                                              // tile i is here for all lanes, tile i - 1 has been read by all
            fetch(i + Cfg::kStages - 1, next);
            next = pages_of(i + Cfg::kStages);
            const int row = begin + (warp + i * kFewWarps) * kTok;
            const uint32_t ks = ring_at + (i % Cfg::kStages) * kStage, vs = ks + kTok * kPitch;
            const uint8_t *ks_p = ring + (i % Cfg::kStages) * kStage;
            const int8_t *ke = reinterpret_cast<const int8_t *>(ks_p + 2 * kTok * kPitch), *ve = ke + kTok;

            // ---- scores of groups of 16 cached rows: rows g8 (elements 0, 1) and g8 + 8 (elements 2, 3) against rows 2c, 2c + 1
            float s[NT][kSubs][4];
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int u = 0; u < kSubs; ++u) s[m][u][0] = s[m][u][1] = s[m][u][2] = s[m][u][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                if (k * 16 < dim) {
#pragma unroll
                    for (int u = 0; u < kSubs; ++u) {
                        uint32_t f[4];
                        if constexpr (!kEight) {
                            ldmatrix4(f, ks + (16 * u + (lane & 15)) * kPitch + k * 32 + (lane >> 4) * 16);
                        } else {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(ks_p + (16 * u + g8) * kPitch + k * 16 + 4 * c4);
                            const uint32_t x = *reinterpret_cast<const uint32_t *>(ks_p + (16 * u + 8 + g8) * kPitch + k * 16 + 4 * c4);
                            f[0] = codes_low(w); f[1] = codes_low(x); f[2] = codes_high(w); f[3] = codes_high(x);
                        }
#pragma unroll
                        for (int m = 0; m < NT; ++m) mma16816<MM>(s[m][u], f, qf[m][k][0], qf[m][k][1]);
                    }
                }
            // ---- scale, mask. `v` is the score with the exponent of its V row added.
            float v[NT][kSubs][4];
#pragma unroll
            for (int u = 0; u < kSubs; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int x = 16 * u + 8 * h + g8;
                    float f = 1.0f, power = 0.0f;
                    if constexpr (kEight) {
                        f = __uint_as_float((uint32_t)(ke[x] + 127) << 23);    // the exponent -128 gives -inf, and a NaN with codes of zero
                        power = ve[x] == kNanExponent ? CUDART_NAN_F : (float)ve[x];
                    }
#pragma unroll
                    for (int m = 0; m < NT; ++m)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            s[m][u][2 * h + j] *= kEight ? f * row_factor[m][j] : row_factor[m][j];
                            v[m][u][2 * h + j] = kEight ? s[m][u][2 * h + j] + power : 0.0f;
                        }
                }
            if (row < full_lo || row + kTok > full_hi || row + kTok > end) {
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = row + 16 * u + 8 * h + g8;
#pragma unroll
                        for (int m = 0; m < NT; ++m)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                if (key >= last[m][j] || key < first[m][j] || key >= end) s[m][u][2 * h + j] = v[m][u][2 * h + j] = -CUDART_INF_F;
                    }
            }
            // ---- weights
            uint32_t pf[NT][kSubs][2];
#pragma unroll
            for (int m = 0; m < NT; ++m) {
                bool moved = false;
                float alpha[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float t4 = -CUDART_INF_F, u4 = -CUDART_INF_F;
#pragma unroll
                    for (int u = 0; u < kSubs; ++u) {
                        t4 = fmaxf(t4, fmaxf(s[m][u][j], s[m][u][2 + j]));
                        if constexpr (kEight) u4 = fmaxf(u4, fmaxf(v[m][u][j], v[m][u][2 + j]));
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        t4 = fmaxf(t4, __shfl_xor_sync(0xFFFFFFFFu, t4, x));
                        if constexpr (kEight) u4 = fmaxf(u4, __shfl_xor_sync(0xFFFFFFFFu, u4, x));
                    }
                    const float now = fmaxf(top[m][j], t4);
                    const float peak = now == -CUDART_INF_F ? 0.0f : now;      // nothing seen yet: every weight is exp2(-inf) = 0
                    const float fall = exp2_fast(top[m][j] - peak), ref = kEight ? peak : peak - kLift;
                    if constexpr (!kEight) moved |= now != top[m][j];
                    top[m][j] = now;
                    alpha[j] = fall;
                    float above = ref;
                    if constexpr (kEight) {
                        const float high = fmaxf(base[m][j], u4);
                        above = high == -CUDART_INF_F ? 0.0f : high;
                        alpha[j] = exp2_fast(base[m][j] - above);
                        above -= kLift;
                        moved |= high != base[m][j];
                        base[m][j] = high;
                    }
                    float part = 0.0f;
#pragma unroll
                    for (int u = 0; u < kSubs; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float &p = s[m][u][2 * h + j];
                            p = exp2_fast(p - ref);
                            part += p;
                            if constexpr (kEight) p = exp2_fast(v[m][u][2 * h + j] - above);
                        }
                    sum[m][j] = sum[m][j] * fall + part;
                }
#pragma unroll
                for (int u = 0; u < kSubs; ++u) {
                    pf[m][u][0] = transpose8(pack2_rn<MM>(s[m][u][0], s[m][u][1]));
                    pf[m][u][1] = transpose8(pack2_rn<MM>(s[m][u][2], s[m][u][3]));
                }
                if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                    for (int n = 0; n < kSteps; ++n) {
                        acc[m][n][0] *= alpha[0]; acc[m][n][1] *= alpha[1];
                        acc[m][n][2] *= alpha[0]; acc[m][n][3] *= alpha[1];
                    }
                }
            }
            // ---- V^T times the weights, 16 elements at a time
#pragma unroll
            for (int n = 0; n < kSteps; ++n)
                if (n * 16 < dim) {
#pragma unroll
                    for (int u = 0; u < kSubs; ++u) {
                        if constexpr (!kEight) {
                            uint32_t f[4];     // rows 0-7 of elements 0-7 and 8-15, then rows 8-15
                            ldmatrix4_trans(f, vs + (16 * u + (lane & 7) + (lane >> 4) * 8) * kPitch + n * 32 + ((lane >> 3) & 1) * 16);
#pragma unroll
                            for (int m = 0; m < NT; ++m) mma16816<MM>(acc[m][n], f, pf[m][u][0], pf[m][u][1]);
                        } else if ((n & 1) == 0) {
                            // pairs of codes travel as 16-bit elements: a word comes back as two neighbours of row 2c and two of row
                            // 2c + 1. The even elements of 16 are the first eight rows of the product, the odd ones the others.
                            const bool two = (n + 1) * 16 < dim;
                            uint32_t f[4];     // rows 0-7 and 8-15 of 16 elements, and of the 16 behind them
                            ldmatrix4_trans(f, vs + (16 * u + (lane & 15)) * kPitch + (two ? n + (lane >> 4) : n) * 16);
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (n + h < kSteps && (h == 0 || two)) {
                                    const uint32_t a0 = codes_low(f[2 * h]), a1 = codes_high(f[2 * h]);
                                    const uint32_t b0 = codes_low(f[2 * h + 1]), b1 = codes_high(f[2 * h + 1]);
                                    const uint32_t g[4] = {__byte_perm(a0, a1, 0x5410), __byte_perm(a0, a1, 0x7632),
                                                           __byte_perm(b0, b1, 0x5410), __byte_perm(b0, b1, 0x7632)};
#pragma unroll
                                    for (int m = 0; m < NT; ++m) mma16816<MM>(acc[m][(n + h) % kSteps], g, pf[m][u][0], pf[m][u][1]);
                                }
                        }
                    }
                }
        }
        copy_wait<0>();

        // ---- the warps' parts meet: [warp][row][maximum, sum, base] and [warp][row][element]
        __syncthreads();
        float4 *stat = reinterpret_cast<float4 *>(smem);
        float *part = reinterpret_cast<float *>(stat + kFewWarps * kRows);
        constexpr int kPart = DPAD + 4;
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float l = sum[m][j];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
                const int r = m * 8 + 2 * c4 + j;
                if (r < t.rows) {
                    if constexpr (!kEight) l *= pow2f(-(int)kLift);
                    if (g8 == 0) stat[warp * kRows + r] = make_float4(top[m][j], l, (kEight ? base[m][j] : top[m][j]) - kLift, 0.0f);
                    float *dst = part + (warp * kRows + r) * kPart;
#pragma unroll
                    for (int n = 0; n < kSteps; ++n) {
                        dst[16 * n + (kEight ? 2 * g8 : g8)] = acc[m][n][j];
                        dst[16 * n + (kEight ? 2 * g8 + 1 : g8 + 8)] = acc[m][n][2 + j];
                    }
                }
            }
        __syncthreads();
        const int64_t heads = a.q.heads;
        const int pitch = dim + 4;
        auto finish = [&](int r, float m, float l, float4 o) {         // a row's output, from this lane's four elements, and its lse
            const int token = token_of(r), qh = head * a.group + (r - token * a.group);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t to = t.q_begin + token;
            uint16_t *dst = reinterpret_cast<uint16_t *>(a.out.p) + to * a.out.token_stride + qh * a.out.head_stride + lane * 4;
            if (lane * 4 < dim) *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2_rn<DT>(o.x * inv, o.y * inv), pack2_rn<DT>(o.z * inv, o.w * inv));
            if (lane == 0 && a.lse) a.lse[to * heads + qh] = l == 0.0f ? -CUDART_INF_F : (m + log2f(l)) * kLn2;
        };
        // a CTA leaves two parts at most: the end of a pair that began before it, and the beginning of one that goes on behind it;
        // [CTA][end, beginning][row][maximum, sum, -, -, elements]
        auto part_at = [&](int cta, bool beginning, int r) { return a.partial + ((int64_t)(2 * cta + (beginning ? 1 : 0)) * few_rows + r) * pitch; };
        auto gather = [&](int r, float &m, float &l, float4 &o) {      // what the warps have in shared memory for a row
            float w[kFewWarps];
            m = -CUDART_INF_F; l = 0.0f;
#pragma unroll
            for (int i = 0; i < kFewWarps; ++i) m = fmaxf(m, stat[i * kRows + r].x);
            const float ref = m == -CUDART_INF_F ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < kFewWarps; ++i) {
                const float4 x = stat[i * kRows + r];
                l = fmaf(exp2_fast(x.x - ref), x.y, l);
                w[i] = exp2_fast(x.z - ref);                           // back from the output's own reference
            }
            o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (lane * 4 < dim) {
#pragma unroll
                for (int i = 0; i < kFewWarps; ++i) {
                    const float4 x = *reinterpret_cast<const float4 *>(part + (i * kRows + r) * kPart + lane * 4);
                    o.x = fmaf(w[i], x.x, o.x); o.y = fmaf(w[i], x.y, o.y); o.z = fmaf(w[i], x.z, o.z); o.w = fmaf(w[i], x.w, o.w);
                }
            }
        };
        for (int r = warp; r < t.rows; r += kFewWarps) {
            float m, l;
            float4 o;
            gather(r, m, l, o);
            if (used == 1) { finish(r, m, l, o); continue; }
            float *p = part_at(blockIdx.x, first_cta == (int)blockIdx.x, r);
            if (lane * 4 < dim) *reinterpret_cast<float4 *>(p + 4 + lane * 4) = o;
            if (lane == 0) *reinterpret_cast<float2 *>(p) = make_float2(m, l);
        }
        // ---- the last of the parts to get here joins them, in their order, so that results are the same from call to call
        if (used > 1) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                int *count = a.arrived + first_cta;                    // at most one pair begins in a CTA and ends in another
                is_last = atomicAdd(count, 1) == used - 1;
                if (is_last) *count = 0;                               // as the next launch expects it
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                // each warp takes every fourth part of a row; [warp][row][maximum, sum] and [warp][row][element] in shared memory, which
                // the parts' reading left free
                const int64_t step = (int64_t)2 * few_rows * pitch;
                for (int r = 0; r < t.rows; ++r) {
                    const float *p0 = part_at(first_cta, true, r), *p1 = part_at(first_cta + 1, false, r) - step;
                    float m = -CUDART_INF_F, l = 0.0f;
                    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int i = warp; i < used; i += kFewWarps) {
                        const float *p = i == 0 ? p0 : p1 + i * step;
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p));
                        const float4 x = lane * 4 < dim ? __ldcg(reinterpret_cast<const float4 *>(p + 4 + lane * 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        const float now = fmaxf(m, ml.x), ref = now == -CUDART_INF_F ? 0.0f : now;
                        const float fall = exp2_fast(m - ref), w = exp2_fast(ml.x - ref);
                        m = now;
                        l = fmaf(l, fall, w * ml.y);
                        o.x = fmaf(o.x, fall, w * x.x); o.y = fmaf(o.y, fall, w * x.y); o.z = fmaf(o.z, fall, w * x.z); o.w = fmaf(o.w, fall, w * x.w);
                    }
                    if (lane == 0) stat[warp * kRows + r] = make_float4(m, l, m, 0.0f);
                    if (lane * 4 < dim) *reinterpret_cast<float4 *>(part + (warp * kRows + r) * kPart + lane * 4) = o;
                }
                __syncthreads();
                for (int r = warp; r < t.rows; r += kFewWarps) {
                    float m, l;
                    float4 o;
                    gather(r, m, l, o);
                    finish(r, m, l, o);
                }
            }
        }
        // ---- on to the next pair
        pair += n;
        at = pair;
        if (at >= until) return;
        if (++head == kv_heads) {
            head = 0;
            do {
                if (++b >= a.batch.batch) return;                       // there is one: the piece goes on
                n = groups_of(a, b, few_rows, t);
            } while (n == 0);
        }
        __syncthreads();                                                // shared memory is free again
    }
}

// `beside`: behind the many-row kernel of the same call, which lets this one start once what came before both is complete. They share
// nothing, so it only waits before it ends, for whoever waits for it.
template <int DT, bool kEight, int DPAD, int NT>
__global__ void __launch_bounds__(kFewThreads, FewCfg<kEight, NT>::kPerSm)
attend_few_kernel(const __grid_constant__ AttentionArgs a, int few_rows, int least, int beside) {
    if (!beside) wait_for_predecessor();
    attend_few<DT, kEight, DPAD, NT>(a, few_rows, least);
    if (beside) wait_for_predecessor();
}

template <int DT, bool kEight, int DPAD, int NT> int launch_few(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early) {
    constexpr int kSmem = FewCfg<kEight, NT>::smem_bytes(DPAD);
    if (int rc = opt_in_shared<attend_few_kernel<DT, kEight, DPAD, NT>, kSmem>()) return rc;
    return launch_kernel(attend_few_kernel<DT, kEight, DPAD, NT>, dim3((unsigned)p.few_ctas), kFewThreads, kSmem, st, early, a, p.few_rows, p.few_least, (int)(p.many_tiles > 0));
}
template <int DT, bool kEight, int DPAD> int launch_few_rows(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early) {
    if (p.few_tile == 8) return launch_few<DT, kEight, DPAD, 1>(a, p, st, early);
    return launch_few<DT, kEight, DPAD, 2>(a, p, st, early);
}
template <int DT, bool kEight> int launch_few_dim(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early) {
    return a.cache.dim <= 64 ? launch_few_rows<DT, kEight, 64>(a, p, st, early) : launch_few_rows<DT, kEight, 128>(a, p, st, early);
}
template <int DT> int launch_all(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early) {
    AttentionArgs many = a;
    const size_t few_bytes = (size_t)2 * p.few_ctas * p.few_rows * (a.cache.dim + 4) * sizeof(float);    // the streaming kernel's parts
    many.partial = a.partial + few_bytes / sizeof(float);
    many.partial_bytes = a.partial_bytes - few_bytes;
    int rc = MAGB200_OK;
    if (p.many_tiles > 0) rc = launch_attend_many(many, p, st, early);
    if (!rc && p.few_ctas > 0) {
        if (p.many_tiles > 0) early = true;                         // behind a kernel of this call
        rc = a.cache.bits == 8 ? launch_few_dim<DT, true>(a, p, st, early) : launch_few_dim<DT, false>(a, p, st, early);
    }
    if (!rc && p.many_tiles > 0) rc = launch_join_many(many, p, st);
    return rc;
}

}  // namespace

size_t attention_workspace_bytes() { return (size_t)64 << 20; }

static int few_places(int tile, int bits) {
    if (tile == 16) return bits == 8 ? FewCfg<true, 2>::kPerSm : FewCfg<false, 2>::kPerSm;
    return bits == 8 ? FewCfg<true, 1>::kPerSm : FewCfg<false, 1>::kPerSm;
}

constexpr int kMostFewRows = 16;
AttentionPlan plan_attention(const KvCache &c, const KvBatch &b, int heads, bool causal, int64_t window, int sms) {
    AttentionPlan p;
    memset(&p, 0, sizeof(p));
    const int64_t group = heads / c.kv_heads, rows = b.max_q * group;
    int64_t keys = b.max_kv < INT32_MAX ? b.max_kv : INT32_MAX; // cached rows that one row tile sees at most
    if (causal && window > 0 && window + b.max_q + 15 < keys) keys = window + b.max_q + 15;
    // A warp tile of the streaming form holds 8 or 16 rows; sequences of more rows than that use the tensor cores' tiles. In a mixed
    // batch the tile is made for the sequences with a single new token. Measured with 8 KV heads of 128, in us (6 sequences on up to
    // 50000 rows, 16 and 8 bits; one sequence on 16000 rows of 16 bits):
    //    8 rows:  in tiles of 8 134, 92 and 27, of 16 136, 121 and 30, on the tensor cores 297, 480 and 35
    //   16 rows:  in tiles of 16 149, 135 and 42, on the tensor cores 297, 479 and 35
    //   32 rows:  in tiles of 32, which spilled registers, 363, 431 and 75, on the tensor cores 299, 484 and 35
    // (64 sequences on up to 4096 rows, 32 rows: 393 and 467 in tiles, 239 and 357 on the tensor cores).
    const int64_t fit = rows <= kMostFewRows ? rows : group;
    p.few_tile = fit <= 8 ? 8 : 16;
    p.few_rows = p.few_tile;
    if (rows <= kMostFewRows || (b.batch > 1 && group <= kMostFewRows)) {
        // one CTA for every place on the multiprocessors, fewer where there is not enough for pieces of 128 cached rows
        const int64_t pieces = c.kv_heads * ((keys + 127) / 128 + 1), places = (int64_t)few_places(p.few_tile, c.bits) * sms;
        p.few_ctas = (int)(pieces < places && b.batch * pieces < places ? b.batch * pieces : places);
        if (p.few_ctas > kMaxFewCtas) p.few_ctas = kMaxFewCtas;
        // a longer line of groups is worth larger pieces: n / p groups to stream against p parts to join, at about 0.16 us each, are
        // least at n / p = sqrt(n) (20000 rows of one head: 31 us with 84 parts, 24 with 36)
        p.few_least = (int)sqrt((double)((keys + 15) / 16));
        if (p.few_least < 8) p.few_least = 8;
    } else {
        p.few_rows = 0;
    }
    if (rows > p.few_rows) {
        p.many_tiles = b.tokens * group / 256 + b.batch;
        p.many_keys = keys;
    }
    return p;
}

int launch_paged_attention(const AttentionArgs &a, cudaStream_t st, bool early) {
    const AttentionPlan p = plan_attention(a.cache, a.batch, a.q.heads, a.causal != 0, a.window, num_sms());
    if (a.batch.max_q * a.group > 0x7FFFF000 || a.batch.tokens * a.q.heads > 0x7FFFF000 ||
        p.many_tiles * a.cache.kv_heads > 1 << 30) {
        set_error("paged_attention: %d sequences of %d KV heads are too many for one launch", a.batch.batch, a.cache.kv_heads);
        return MAGB200_ERR_TOO_LARGE;
    }
    return a.cache.dtype == MAGB200_BF16 ? launch_all<MAGB200_BF16>(a, p, st, early) : launch_all<MAGB200_F16>(a, p, st, early);
}

}  // namespace magb200
