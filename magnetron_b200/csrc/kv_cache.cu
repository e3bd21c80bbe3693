// The passes around attention that move each byte once: head norm + rotation of q and k, the paged KV cache as it is
// written and as it is read back. All are bound by HBM for long batches and by a launch's latency for a decode step, so each is
// one launch without a workspace; a row (one head of one token) belongs to a group of lanes, eight elements each in
// the first and sixteen in the others.
#include "attention.cuh"

namespace magb200 {
namespace {

constexpr int kRowThreads = 256;

// ---- eight elements of a row ----------------------------------------------------------------------------------------------
template <int DT> struct Eight;   // raw bits of eight elements
template <> struct Eight<MAGB200_F32> { uint4 a, b; };
template <> struct Eight<MAGB200_F16> { uint4 a; };
template <> struct Eight<MAGB200_BF16> { uint4 a; };

template <int DT> __device__ __forceinline__ void to_floats(const Eight<DT> &r, float (&x)[8]) {
    if constexpr (DT == MAGB200_F32) {
        x[0] = __uint_as_float(r.a.x); x[1] = __uint_as_float(r.a.y); x[2] = __uint_as_float(r.a.z); x[3] = __uint_as_float(r.a.w);
        x[4] = __uint_as_float(r.b.x); x[5] = __uint_as_float(r.b.y); x[6] = __uint_as_float(r.b.z); x[7] = __uint_as_float(r.b.w);
    } else {
        unpack2<DT>(r.a.x, x[0], x[1]); unpack2<DT>(r.a.y, x[2], x[3]);
        unpack2<DT>(r.a.z, x[4], x[5]); unpack2<DT>(r.a.w, x[6], x[7]);
    }
}
template <int DT> __device__ __forceinline__ Eight<DT> from_floats(const float (&x)[8]) {
    Eight<DT> r;
    if constexpr (DT == MAGB200_F32) {
        r.a = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        r.b = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
    } else {
        r.a = make_uint4(pack2_rn<DT>(x[0], x[1]), pack2_rn<DT>(x[2], x[3]), pack2_rn<DT>(x[4], x[5]), pack2_rn<DT>(x[6], x[7]));
    }
    return r;
}
// `vec`: the address is on a 16-byte boundary
template <int DT> __device__ __forceinline__ Eight<DT> load8(const void *p, int64_t at, bool vec) {
    Eight<DT> r;
    if constexpr (DT == MAGB200_F32) {
        const uint32_t *s = reinterpret_cast<const uint32_t *>(p) + at;
        if (vec) { r.a = *reinterpret_cast<const uint4 *>(s); r.b = *reinterpret_cast<const uint4 *>(s + 4); }
        else { r.a = make_uint4(s[0], s[1], s[2], s[3]); r.b = make_uint4(s[4], s[5], s[6], s[7]); }
    } else {
        const uint16_t *s = reinterpret_cast<const uint16_t *>(p) + at;
        if (vec) r.a = *reinterpret_cast<const uint4 *>(s);
        else r.a = make_uint4(s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16, s[4] | (uint32_t)s[5] << 16, s[6] | (uint32_t)s[7] << 16);
    }
    return r;
}
template <int DT> __device__ __forceinline__ void store8(void *p, int64_t at, const Eight<DT> &r, bool vec) {
    if constexpr (DT == MAGB200_F32) {
        uint32_t *s = reinterpret_cast<uint32_t *>(p) + at;
        if (vec) { *reinterpret_cast<uint4 *>(s) = r.a; *reinterpret_cast<uint4 *>(s + 4) = r.b; }
        else { s[0] = r.a.x; s[1] = r.a.y; s[2] = r.a.z; s[3] = r.a.w; s[4] = r.b.x; s[5] = r.b.y; s[6] = r.b.z; s[7] = r.b.w; }
    } else {
        uint16_t *s = reinterpret_cast<uint16_t *>(p) + at;
        if (vec) *reinterpret_cast<uint4 *>(s) = r.a;
        else {
            s[0] = (uint16_t)r.a.x; s[1] = (uint16_t)(r.a.x >> 16); s[2] = (uint16_t)r.a.y; s[3] = (uint16_t)(r.a.y >> 16);
            s[4] = (uint16_t)r.a.z; s[5] = (uint16_t)(r.a.z >> 16); s[6] = (uint16_t)r.a.w; s[7] = (uint16_t)(r.a.w >> 16);
        }
    }
}
template <int DT> struct Sixteen { Eight<DT> a, b; };
bool rows_on_16(const HeadRows &r, size_t es) {
    return ((uintptr_t)r.p & 15u) == 0 && (r.token_stride * (int64_t)es) % 16 == 0 && (r.head_stride * (int64_t)es) % 16 == 0;
}

// ---- head norm + rotation -------------------------------------------------------------------------------------------------
// y = x * rsqrt(mean(x^2) + eps) * w, then (a, b) -> (a c - b s, a s + b c) for the pairs of the first `rotary` elements, where
// c, s = factor * cos, sin(position * inv_freq[i]). Everything in fp32 with one rounding at the end, except the angle: at
// position 2^17 an fp32 product would be off by 2^-7 rad, so the turns (angle / 2 pi) are formed and reduced in fp64 and only
// the fraction goes to the fp32 sine. A token's rotary/2 sines are made once, in shared memory, and used by all its heads.
// One lane holds eight elements as four pairs: of the half layout elements 4u..4u+3 and the same of the second half, of the
// interleaved layout and of the part that is not turned eight neighbours. The sum of squares does not care.
struct NormRopeArgs {
    HeadRows q, k, q_out, k_out;
    const void *q_weight, *k_weight;
    RopeArgs rope;
    float eps;
    int dim;
    int64_t tokens;
    int vec, per_cta;
};
// Where pair p (0 .. dim/2) of a row has its two elements.
__device__ __forceinline__ int2 pair_at(int p, int rotary, int interleaved) {
    const int half = rotary >> 1;
    if (p < half && !interleaved) return make_int2(p, p + half);
    return make_int2(2 * p, 2 * p + 1);
}
// A lane's elements are kRun pairs. kVec: two runs of kRun at `o0` and `o1`, on boundaries of kRun elements; `apart`: a pair has
// one element in each run, otherwise its two are neighbours in one. Without kVec they come element by element, always apart.
struct Place { int o0, o1; bool apart; };
template <int DT> __device__ __forceinline__ void load_run(const void *p, int64_t at, float (&x)[4]) {
    if constexpr (DT == MAGB200_F32) {
        const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(p) + at);
        unpack2<DT>(v.x, x[0], x[1]); unpack2<DT>(v.y, x[2], x[3]);
    }
}
template <int DT> __device__ __forceinline__ void load_run(const void *p, int64_t at, float (&x)[8]) { to_floats<DT>(load8<DT>(p, at, true), x); }
template <int DT> __device__ __forceinline__ void store_run(void *p, int64_t at, const float (&x)[4]) {
    if constexpr (DT == MAGB200_F32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p) + at) = make_uint2(pack2_rn<DT>(x[0], x[1]), pack2_rn<DT>(x[2], x[3]));
}
template <int DT> __device__ __forceinline__ void store_run(void *p, int64_t at, const float (&x)[8]) { store8<DT>(p, at, from_floats<DT>(x), true); }
template <int DT, int kRun, bool kVec>
__device__ __forceinline__ void load_runs(const void *base, int64_t row, int u, const RopeArgs &r, const Place &at, float (&a)[kRun], float (&b)[kRun]) {
    if constexpr (kVec) {
        load_run<DT>(base, row + at.o0, a);
        load_run<DT>(base, row + at.o1, b);
    } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int2 p = pair_at(kRun * u + i, r.rotary, r.interleaved);
            a[i] = load_as_f32<DT>(base, row + p.x);
            b[i] = load_as_f32<DT>(base, row + p.y);
        }
    }
}

// A CTA takes up to kTurnTokens tokens: their sines are one round of its threads, so that the chain position -> fp64 -> sine ->
// barrier is paid once for all of them, and their rows follow in one stream. A row of 128 is 16 lanes' worth of a hundred
// instructions, so what a lane needs of its place is settled before the loop; even so 53 % of the issue slots are taken, and the 27 warps
// of a multiprocessor (63 registers a thread) wait for their rows most of the rest (8192 tokens of 72 heads: 68 us, 0.68 of the copy rate).
constexpr int kTurnTokens = 4;
template <int DT, int LPR, int kRun, bool kVec>
__global__ void __launch_bounds__(kRowThreads, 4) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
    __shared__ __align__(16) float2 turn[kTurnTokens][128];        // factor * (cos, sin) of each pair; dim <= 256
    constexpr int kGroups = kRowThreads / LPR;
    wait_for_predecessor();
    const int u = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int half = a.rope.rotary >> 1;
    const bool mine = 2 * kRun * u < a.dim;
    Place at;
    at.apart = !kVec || (!a.rope.interleaved && kRun * u < half);
    at.o0 = at.apart ? kRun * u : 2 * kRun * u;
    at.o1 = at.apart ? kRun * u + half : 2 * kRun * u + kRun;
    const int64_t first = (int64_t)blockIdx.x * a.per_cta;
    const int tokens = (int)(a.tokens - first < a.per_cta ? a.tokens - first : a.per_cta);
    for (int i = threadIdx.x; i < half * tokens; i += kRowThreads) {
        const int token = i / half, pair = i - token * half;
        const double turns = (double)a.rope.positions[first + token] * (double)a.rope.inv_freq[pair] * 0.15915494309189535;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[token][pair] = make_float2(a.rope.factor * c, a.rope.factor * s);
    }
    __syncthreads();
    const float inv_dim = 1.0f / (float)a.dim;
    // a group of LPR lanes has one row, so its lanes are at the shuffles together
    const uint32_t lanes = LPR == 32 ? 0xFFFFFFFFu : ((1u << (LPR & 31)) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
    auto side = [&](const HeadRows &src, const HeadRows &dst, const void *weight) {
        if (src.heads == 0) return;
        float ga[kRun], gb[kRun];
        if (mine && weight) load_runs<DT, kRun, kVec>(weight, 0, u, a.rope, at, ga, gb);
        const int n = blockIdx.y * kGroups + group;
        const int step = kGroups * gridDim.y, step_tokens = step / src.heads, step_heads = step - step_tokens * src.heads;
        int token = n / src.heads, h = n - token * src.heads;
        while (token < tokens) {
            float xa[kRun], xb[kRun];
#pragma unroll
            for (int j = 0; j < kRun; ++j) xa[j] = xb[j] = 0.0f;
            if (mine) load_runs<DT, kRun, kVec>(src.p, (first + token) * src.token_stride + h * src.head_stride, u, a.rope, at, xa, xb);
            if (weight) {
                auto mean = [&](float by, float eps) {                     // of the squares of by * x, over all the row's lanes, and eps
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < kRun; ++j) {
                        const float p = xa[j] * by, q = xb[j] * by;
                        sum = fmaf(p, p, fmaf(q, q, sum));
                    }
#pragma unroll
                    for (int m = LPR / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(lanes, sum, m);
                    return fmaf(sum, inv_dim, eps);
                };
                const float square = mean(1.0f, a.eps);
                float inv = rsqrtf(square);
                // squares past the range of fp32, or so small that they lose bits, are taken again of the row times a power of two; it goes
                // to the root of large rows and to the elements of small ones, which loses nothing of either
                if (!(square >= 0x1p-100f && square <= 3.4028235e38f)) {
                    const bool small = square < 1.0f;
                    const float by = small ? 0x1p96f : 0x1p-70f;
                    inv = rsqrtf(mean(by, a.eps * by * by));
                    if (!small) inv *= by;
#pragma unroll
                    for (int j = 0; j < kRun; ++j)
                        if (small) { xa[j] *= by; xb[j] *= by; }
                }
                if (mine) {
#pragma unroll
                    for (int j = 0; j < kRun; ++j) { xa[j] = xa[j] * inv * ga[j]; xb[j] = xb[j] * inv * gb[j]; }
                }
            }
            if (kRun * u < half) {
                const float2 *cs = &turn[token][kRun * u];
                if (at.apart) {
#pragma unroll
                    for (int j = 0; j < kRun; ++j)
                        if (kVec || kRun * u + j < half) {
                            const float p = xa[j], q = xb[j];
                            xa[j] = p * cs[j].x - q * cs[j].y;
                            xb[j] = fmaf(p, cs[j].y, q * cs[j].x);
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < kRun; j += 2) {
                        const float2 ca = cs[j >> 1], cb = cs[(kRun + j) >> 1];
                        const float p = xa[j], q = xa[j + 1], v = xb[j], w = xb[j + 1];
                        xa[j] = p * ca.x - q * ca.y;
                        xa[j + 1] = fmaf(p, ca.y, q * ca.x);
                        xb[j] = v * cb.x - w * cb.y;
                        xb[j + 1] = fmaf(v, cb.y, w * cb.x);
                    }
                }
            }
            if (mine) {
                const int64_t to = (first + token) * dst.token_stride + h * dst.head_stride;
                if constexpr (kVec) {
                    store_run<DT>(dst.p, to + at.o0, xa);
                    store_run<DT>(dst.p, to + at.o1, xb);
                } else {
#pragma unroll
                    for (int j = 0; j < kRun; ++j) {
                        const int2 p = pair_at(kRun * u + j, a.rope.rotary, a.rope.interleaved);
                        store_from_f32<DT>(dst.p, to + p.x, xa[j]);
                        store_from_f32<DT>(dst.p, to + p.y, xb[j]);
                    }
                }
            }
            h += step_heads;
            token += step_tokens;
            if (h >= src.heads) { h -= src.heads; ++token; }
        }
    };
    side(a.q, a.q_out, a.q_weight);
    side(a.k, a.k_out, a.k_weight);
}

template <int DT> int launch_norm_rope_dt(const NormRopeArgs &a, cudaStream_t st, bool early) {
    // sixteen elements a lane where the row's runs allow it (8192 tokens of 72 heads of 128: 75 us with eight), else eight
    const bool wide = a.vec && a.rope.rotary % 16 == 0 && a.dim % 16 == 0;
    const int per_lane = wide ? 16 : 8;
    const int lpr = a.dim <= 8 * per_lane ? 8 : a.dim <= 16 * per_lane ? 16 : 32;
    const int rows = a.q.heads + a.k.heads, groups = kRowThreads / lpr;
    const int passes = (rows + groups - 1) / groups;
    NormRopeArgs n = a;
    const int64_t spread = a.tokens / ((int64_t)num_sms() * 4);
    n.per_cta = (int)(spread < 1 ? 1 : spread > kTurnTokens ? kTurnTokens : spread);
    // few tokens: spread a token's heads over CTAs as well, so that no CTA walks rows one after another
    const int64_t room = (int64_t)num_sms() * 8 / a.tokens;
    const dim3 grid((unsigned)((a.tokens + n.per_cta - 1) / n.per_cta), (unsigned)(room < 1 ? 1 : room < passes ? room : passes));
    auto run = [&](auto *kernel) { return launch_kernel(kernel, grid, kRowThreads, 0, st, early, n); };
    if (wide) return lpr == 8 ? run(qk_norm_rope_kernel<DT, 8, 8, true>) : run(qk_norm_rope_kernel<DT, 16, 8, true>);
    if (a.vec) return lpr == 8 ? run(qk_norm_rope_kernel<DT, 8, 4, true>) : lpr == 16 ? run(qk_norm_rope_kernel<DT, 16, 4, true>) : run(qk_norm_rope_kernel<DT, 32, 4, true>);
    return lpr == 8 ? run(qk_norm_rope_kernel<DT, 8, 4, false>) : lpr == 16 ? run(qk_norm_rope_kernel<DT, 16, 4, false>) : run(qk_norm_rope_kernel<DT, 32, 4, false>);
}

// ---- cache write / read ---------------------------------------------------------------------------------------------------
// A CTA takes `per_cta` tokens: its warps find each token's sequence, page and slot once, then groups of lanes move the
// token's 2 * kv_heads rows.
constexpr int kMaxTokensPerCta = 16;
struct Slot { int64_t page; int offset; };   // page < 0: nothing to do for this token

// The page and slot of position `pos` of sequence b. Bounds are checked here: what does not fit raises the word and is skipped.
__device__ __forceinline__ Slot locate(const KvCache &c, const KvBatch &b, int seq, int64_t pos) {
    Slot s;
    s.page = -1;
    s.offset = (int)(pos & (c.page_size - 1));
    if (pos < 0) return s;                    // fewer cached tokens than new ones: this one has no place
    const int64_t entry = pos >> c.page_shift;
    if (entry >= b.max_pages) { atomicOr(b.status + kBatchWord, kBadLength); return s; }
    const int32_t page = b.table[(int64_t)seq * b.max_pages + entry];
    if (page < 0 || page >= c.pages) { atomicOr(b.status + kBatchWord, kBadPage); return s; }
    s.page = page;
    return s;
}

// Whether the offsets of a sequence fit: they ascend, stay within the rows and, of a write, hold at most max_q new tokens.
template <bool kRead> __device__ __forceinline__ bool offsets_fit(const KvBatch &b, int64_t begin, int64_t end) {
    return begin >= 0 && end >= begin && end <= b.tokens && (kRead || end - begin <= b.max_q);
}
// The threads of the grid look at all sequences' offsets, those that no token leads to among them. A function of its own: inside the
// kernel it costs the moves behind it their schedule (write of 32768 tokens to 8 bits 42.5 us, so 45 to 46).
template <bool kRead> __device__ __noinline__ void check_offsets(const KvBatch &b, const int32_t *cu) {
    for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < b.batch; i += (int64_t)gridDim.x * kRowThreads)
        if (!offsets_fit<kRead>(b, cu[i], cu[i + 1])) atomicOr(b.status + kBatchWord, kBadRows);
}

struct CacheMoveArgs {
    KvCache cache;
    KvBatch batch;
    const int32_t *cu;        // offsets of the sequences in the packed rows: cu_q (write) or cu_kv (read)
    HeadRows k, v;
    int per_cta;
    int vec;
};

template <int DT, int LPR, bool kRead, bool kEight>
__global__ void __launch_bounds__(kRowThreads) kv_move_kernel(const __grid_constant__ CacheMoveArgs a) {
    __shared__ Slot slots[kMaxTokensPerCta];
    constexpr int kGroups = kRowThreads / LPR;
    wait_for_predecessor();
    const int64_t first = (int64_t)blockIdx.x * a.per_cta;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const KvCache &c = a.cache;
    if (blockIdx.x <= (unsigned)a.batch.batch / kRowThreads) check_offsets<kRead>(a.batch, a.cu);
    for (int i = warp; i < a.per_cta; i += kRowThreads / 32) {
        const int64_t t = first + i;
        Slot s;
        s.page = -1; s.offset = 0;
        if (t < a.batch.tokens) {
            const int seq = find_sequence(a.cu, a.batch.batch, t, lane);
            const int64_t begin = a.cu[seq], end = a.cu[seq + 1], kv = a.batch.kv_len[seq];
            // rows behind the last sequence belong to nobody; those of one whose offsets do not fit (offsets_fit) are not moved
            if (t >= begin && t < end && begin >= 0 && end <= a.batch.tokens && (kRead || end - begin <= a.batch.max_q)) {
                const int64_t pos = kRead ? t - begin : kv - (end - t);
                if (lane == 0) {
                    if (kRead && pos >= kv) atomicOr(a.batch.status + kBatchWord, kBadLength);   // more rows asked for than are cached
                    else if (!kRead && kv < 0) atomicOr(a.batch.status + kBatchWord, kBadLength);
                    else s = locate(c, a.batch, seq, pos);
                }
            }
        }
        if (lane == 0) slots[i] = s;
    }
    __syncthreads();
    const int u = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const bool mine = 16 * u < c.dim;
    const unsigned rows = 2u * (unsigned)c.kv_heads, total = rows * (unsigned)a.per_cta;
    // kBatch rows of a group are loaded before the first is used; all lanes of a warp go round together (us with one and
    // with two: 16-bit write of 32768 tokens 48.7 and 45.8, 16-bit read of long sequences 122.1 and 119.2, 8-bit read 99.0 and 97.7). A
    // write to 8 bits has too much to do per row (42.7 and 49): quantising takes 74 % of the issue slots, the integer pipe is busy 69 % of
    // the time.
    constexpr int kBatch = !kEight || kRead ? 2 : 1;
    for (unsigned base = 0; base < total; base += kBatch * kGroups) {
        int64_t row[kBatch], cell[kBatch];    // element of the packed rows, row of the cache (-1: nothing to do)
        bool is_v[kBatch];
        Sixteen<DT> x[kBatch];
        uint4 codes[kBatch];
        int e[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const unsigned r = base + j * kGroups + group, i = r / rows, rest = r - i * rows;
            cell[j] = -1;
            is_v[j] = rest >= (unsigned)c.kv_heads;
            x[j].a.a = x[j].b.a = codes[j] = make_uint4(0u, 0u, 0u, 0u);
            e[j] = 0;
            if (r >= total) continue;
            const Slot s = slots[i];
            if (s.page < 0) continue;
            const int h = (int)(is_v[j] ? rest - c.kv_heads : rest);
            const HeadRows &side = is_v[j] ? a.v : a.k;
            row[j] = (first + i) * side.token_stride + h * side.head_stride + 16 * u;
            cell[j] = (s.page * c.kv_heads + h) * c.page_size + s.offset;
            const uint8_t *pool = is_v[j] ? c.v : c.k;
            if (!mine) continue;
            if constexpr (!kRead) {
                x[j].a = load8<DT>(side.p, row[j], a.vec != 0);
                x[j].b = load8<DT>(side.p, row[j] + 8, a.vec != 0);
            } else if constexpr (!kEight) {
                const uint4 *at = reinterpret_cast<const uint4 *>(pool + (cell[j] * c.dim + 16 * u) * 2);
                x[j].a.a = at[0];
                x[j].b.a = at[1];
            } else {
                e[j] = (is_v[j] ? c.v_exp : c.k_exp)[cell[j]];
                codes[j] = *reinterpret_cast<const uint4 *>(pool + cell[j] * c.dim + 16 * u);
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            uint8_t *pool = is_v[j] ? c.v : c.k;
            const HeadRows &side = is_v[j] ? a.v : a.k;
            const bool live = cell[j] >= 0 && mine;
            if constexpr (!kEight && !kRead) {
                if (!live) continue;
                uint4 *at = reinterpret_cast<uint4 *>(pool + (cell[j] * c.dim + 16 * u) * 2);
                at[0] = x[j].a.a;
                at[1] = x[j].b.a;
            } else if constexpr (kRead) {
                if (!live) continue;
                if constexpr (kEight) {
                    const float scale = row_scale(e[j]);
                    const uint32_t in[4] = {codes[j].x, codes[j].y, codes[j].z, codes[j].w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float f[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float2 v = unpack2_e4m3(in[2 * h + (k >> 1)] >> (16 * (k & 1)));
                            f[2 * k] = v.x * scale;
                            f[2 * k + 1] = v.y * scale;
                        }
                        (h == 0 ? x[j].a : x[j].b) = from_floats<DT>(f);
                    }
                }
                store8<DT>(side.p, row[j], x[j].a, a.vec != 0);
                store8<DT>(side.p, row[j] + 8, x[j].b, a.vec != 0);
            } else {
                // as integers the magnitudes of either type order like the numbers, NaN above infinity: two at a time
                const uint32_t in[8] = {x[j].a.a.x, x[j].a.a.y, x[j].a.a.z, x[j].a.a.w, x[j].b.a.x, x[j].b.a.y, x[j].b.a.z, x[j].b.a.w};
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) top = __vmaxu2(top, in[k] & 0x7FFF7FFFu);
                top = max(top >> 16, top & 0xFFFFu);
#pragma unroll
                for (int m = LPR / 2; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, m));
                const int p = row_exponent(DT == MAGB200_BF16 ? top << 16 : f16_bits_to_f32_bits(top));
                const float inv = p == kNanExponent ? 0.0f : pow2f(-p);
                uint32_t out[4] = {0u, 0u, 0u, 0u};
                if (p != kNanExponent) {
                    const float most = most_code<DT>(p);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        float lo, hi;
                        unpack2<DT>(in[k], lo, hi);
                        // no code passes 448: |x| <= 448 * 2^p. Where 240 is the last finite one the numbers are cut there first.
                        lo *= inv; hi *= inv;
                        if (most < 448.0f) { lo = fminf(fmaxf(lo, -most), most); hi = fminf(fmaxf(hi, -most), most); }
                        out[k >> 1] |= pack2_e4m3(lo, hi) << (16 * (k & 1));
                    }
                }
                if (live) *reinterpret_cast<uint4 *>(pool + cell[j] * c.dim + 16 * u) = make_uint4(out[0], out[1], out[2], out[3]);
                if (cell[j] >= 0 && u == 0) (is_v[j] ? c.v_exp : c.k_exp)[cell[j]] = (int8_t)p;
            }
        }
    }
}

template <int DT, bool kRead, bool kEight> int launch_move(const CacheMoveArgs &a, cudaStream_t st, bool early) {
    const dim3 grid((unsigned)((a.batch.tokens + a.per_cta - 1) / a.per_cta));
    auto run = [&](auto *kernel) { return launch_kernel(kernel, grid, kRowThreads, 0, st, early, a); };
    return a.cache.dim <= 64 ? run(kv_move_kernel<DT, 4, kRead, kEight>) : a.cache.dim <= 128 ? run(kv_move_kernel<DT, 8, kRead, kEight>) : run(kv_move_kernel<DT, 16, kRead, kEight>);
}
template <bool kRead> int launch_move_any(const KvCache &c, const KvBatch &b, const int32_t *cu, const HeadRows &k, const HeadRows &v, cudaStream_t st, bool early) {
    CacheMoveArgs a;
    a.cache = c; a.batch = b; a.cu = cu; a.k = k; a.v = v;
    a.vec = rows_on_16(k, 2) && rows_on_16(v, 2);
    const int64_t spread = b.tokens / ((int64_t)num_sms() * 8);
    a.per_cta = (int)(spread < 1 ? 1 : spread > kMaxTokensPerCta ? kMaxTokensPerCta : spread);
    if (c.dtype == MAGB200_BF16) return c.bits == 8 ? launch_move<MAGB200_BF16, kRead, true>(a, st, early) : launch_move<MAGB200_BF16, kRead, false>(a, st, early);
    return c.bits == 8 ? launch_move<MAGB200_F16, kRead, true>(a, st, early) : launch_move<MAGB200_F16, kRead, false>(a, st, early);
}

}  // namespace

int launch_qk_norm_rope(int dtype, int64_t tokens, int dim, const HeadRows &q, const HeadRows &k, const void *q_weight, const void *k_weight,
                        float eps, const RopeArgs &rope, const HeadRows &q_out, const HeadRows &k_out, cudaStream_t st, bool early) {
    NormRopeArgs a;
    a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out;
    a.q_weight = q_weight; a.k_weight = k_weight;
    a.rope = rope; a.eps = eps; a.dim = dim; a.tokens = tokens;
    const size_t es = dtype_size(dtype);
    // the vector form splits a row into units of four pairs; a rotated part that ends inside a unit takes single elements
    a.vec = rope.rotary % 8 == 0 && rows_on_16(q, es) && rows_on_16(q_out, es) && (k.heads == 0 || (rows_on_16(k, es) && rows_on_16(k_out, es))) &&
            ((uintptr_t)q_weight & 15u) == 0 && ((uintptr_t)k_weight & 15u) == 0;
    switch (dtype) {
        case MAGB200_F32: return launch_norm_rope_dt<MAGB200_F32>(a, st, early);
        case MAGB200_F16: return launch_norm_rope_dt<MAGB200_F16>(a, st, early);
        default: return launch_norm_rope_dt<MAGB200_BF16>(a, st, early);
    }
}
int launch_kv_write(const KvCache &c, const KvBatch &b, const HeadRows &k, const HeadRows &v, cudaStream_t st, bool early) {
    return launch_move_any<false>(c, b, b.cu_q, k, v, st, early);
}
int launch_kv_read(const KvCache &c, const KvBatch &b, const int32_t *cu_kv, const HeadRows &k, const HeadRows &v, cudaStream_t st, bool early) {
    return launch_move_any<true>(c, b, cu_kv, k, v, st, early);
}

}  // namespace magb200
