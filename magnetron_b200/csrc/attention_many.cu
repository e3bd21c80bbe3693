// Attention of many rows (a prompt, a chunk of one): 256 (token, head) rows against the cached rows of one KV head on the
// 5th-generation tensor cores.
//
// One persistent CTA per SM takes pieces of work one after the other -- two tiles of 128 rows and their cached rows or, of the last
// units, a part of them; the longest of a sequence first, from a counter -- and walks the cached rows in blocks of 128:
//   warps 0-3, 4-7 : softmax of tile 0 and tile 1, one row per thread, scores read from TMEM and weights written back to it
//   warps 8-11     : loader of K and V blocks through the block table into a ring of shared-memory buffers
//   warps 12, 14   : one thread each issues the MMAs of one tile (one thread for both spent 5.4 k clocks a block, of which
//                    the softmax warps waited 3 k)
//   warp 13        : hands out the work (warp 15 only completes the warpgroup, for the register split)
// For each tile t and block j:  S_t = Q_t K_j^T (both operands in shared memory, K-major), the softmax warps turn S_t into
// weights P_t in place (16-bit, over the same TMEM columns), O_t += P_t V_j (P from TMEM, V in shared memory as it lies, which is
// MN-major). While tile 0 is in its softmax the tensor cores work for tile 1 and the other way round. TMEM: S_0, S_1 of 128
// columns each, O_0, O_1 of head_dim columns each.
//
// The running maximum is a reference that only moves when a row's maximum has grown by more than 2^8 in its exponentials
// (fp32 sums and 16-bit floats hold that with the same relative error): O is then rescaled in TMEM by the row's thread, between
// its block's scores (complete only after the product before them) and its weights (which the next product waits for), so
// the rescaling needs no barrier of its own.
//
// Work: 4 * 128 * 128 * head_dim flop per tile and block = 1024 clocks of the tensor pipe at head_dim 128, and 16384
// exponentials = 1024 clocks of the special-function unit. Measured: 5200 clocks for a block of both tiles, 39 % of either
// (2368 tokens of 16 heads on 14016 rows, 110 blocks a multiprocessor, without a mask: 310 us at 1.85 GHz, 880 TFLOP/s; over 8-bit rows 372 us
// at 1.97 GHz, 6600 clocks; a prefill of 8 x 2048 tokens under the causal mask: 409 us, 672 TFLOP/s). What bounds it is the chain scores -> maximum -> exponentials -> weights -> product of the two tiles, which fall in step,
// and about 14000 clocks a piece of work beside its blocks. Exponentials by a polynomial on the FMA pipe, a token between the tiles
// and weights in a place of their own (heads of 64: 255 -> 265 us) cost more than they brought.
#include "attention_dev.cuh"
#include "tc_ptx.cuh"

namespace magb200 {
namespace {

constexpr int kManyThreads = 512, kManyRows = 256, kBlock = 128;
constexpr int kLoaders = 128;
// A softmax thread holds the 128 scores of its row. The block starts with 512 * 128 = 65536 registers (the launch bound); the
// shares of the four warpgroups add up to just that: 2 * 184 + 80 + 64 = 4 * 128 a thread.
constexpr int kSoftmaxRegs = 184, kLoaderRegs = 80, kIssuerRegs = 64;
static_assert(2 * kSoftmaxRegs + kLoaderRegs + kIssuerRegs == 4 * 128, "a warpgroup would wait for registers that nobody gives up");
constexpr float kMoveAt = 8.0f;              // exponent of two by which a row's maximum may outgrow its reference
// Exponent by which fp16 weights are scaled up: they reach to 2^15 then, keep all their bits down to 2^-21 of the reference and are off
// by 2^-32 of it at most below that (2^-25 unscaled, which thousands of rows of small weight would miss). With a reference that
// moves at 2^4 and a lift of 11 a mixed batch takes 69.5 us, so 67.8. bf16 has the range of fp32.
template <int DT> constexpr float kLift = DT == MAGB200_F16 ? 7.0f : 0.0f;
constexpr int kTimeoutStatus = 1;
constexpr uint64_t kBlockNs = 20000;         // a block of both tiles takes 2.6 us; eight times that

template <int DPAD, bool kEight> struct ManyCfg {
    static constexpr int kBuffers = DPAD == 128 ? (kEight ? 3 : 4) : 8;
    static constexpr int kBufferBytes = kBlock * DPAD * 2;          // one block of K or V
    static constexpr int kTileBytes = 128 * DPAD * 2;               // queries of one tile
    static constexpr int kTailBytes = 512;                          // work slots, barriers
    static constexpr int kRawBytes = kEight ? kBlock * DPAD : 0;    // one block of codes as they come, two of them
    static constexpr int kPatchBytes = 8 * 4096;                    // a patch of 32 rows of 128 bytes for each softmax warp
    static constexpr int kSmem = 1024 + 2 * kTileBytes + kBuffers * kBufferBytes + 2 * kRawBytes + kPatchBytes + kTailBytes;
    static_assert(kSmem <= 227 * 1024, "shared memory of a multiprocessor");
    static constexpr uint32_t kOutCol = 256;                         // TMEM column of O_0; S_t at 128 t
};

// A 16-byte chunk c of row r of a block or query tile: columns of 64 elements, rows of 128 bytes, chunks XOR-swizzled by row.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)((c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) { tcgen05_mma_f16(d, a, b, idesc, accumulate ? 1u : 0u); }
// A from TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u) : "memory");
}
// Columns of TMEM into registers. The registers are filled when the wait returns; filled_32() stands behind the wait and is what
// the uses depend on, so that none of them is moved ahead of it.
__device__ __forceinline__ void tmem_load_32(uint32_t taddr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void filled_32(float *r) {
    asm volatile("" : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
          "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
          "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
          "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31]));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
template <int N> __device__ __forceinline__ void tmem_load_row(uint32_t taddr, float *r) {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_load_32(taddr + c, r + c);
    tmem_load_wait();
#pragma unroll
    for (int c = 0; c < N; c += 32) filled_32(r + c);
}
__device__ __forceinline__ void tmem_load_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
template <int N> __device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Columns outside from .. to - 1 become -inf.
template <int N> __device__ __forceinline__ void mask_columns(float *x, int from, int to) {
#pragma unroll
    for (int c = 0; c < N; ++c)
        if (c < from || c >= to) x[c] = -CUDART_INF_F;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ void fma2(float &x, float &y, float a, float b) {      // x, y = x * a + b, y * a + b
    asm("{\n\t.reg .b64 v, m, n;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 n, {%3, %3};\n\t"
        "fma.rn.f32x2 v, v, m, n;\n\tmov.b64 {%0, %1}, v;\n\t}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float &x, float &y, float a, float b) {      // x, y += a, b
    asm("{\n\t.reg .b64 v, m;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %3};\n\tadd.rn.f32x2 v, v, m;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 256-row tiles of sequence i; none of the sequences whose rows the other kernel takes.
__device__ __forceinline__ int tiles_of(const AttentionArgs &a, int few_rows, int i) {
    if (i >= a.batch.batch) return 0;
    const int64_t len = (int64_t)a.batch.cu_q[i + 1] - a.batch.cu_q[i], rows = len * a.group;
    if (len < 0 || len > a.batch.max_q) { atomicOr(a.batch.status + kBatchWord, kBadRows); return 0; }
    return rows > few_rows ? (int)((rows + kManyRows - 1) / kManyRows) : 0;
}
// Tiles of all sequences, by a whole warp; `most`: what sound offsets add up to at most.
__device__ __forceinline__ int count_tiles(const AttentionArgs &a, int few_rows, int most, int lane) {
    int64_t n = 0;
    for (int i = lane; i < a.batch.batch; i += 32) n += tiles_of(a, few_rows, i);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, s);
    return n < most ? (int)n : most;
}
// Which sequence and tile number `unit` is: sequences in order, the last tile of each first (under a causal mask it is the
// longest). By a whole warp; false: past the last one.
__device__ __forceinline__ bool find_tile(const AttentionArgs &a, int few_rows, int unit, int lane, int &b, int &tile) {
    int before = 0;
    for (int first = 0; first < a.batch.batch; first += 32) {
        int upto = tiles_of(a, few_rows, first + lane);
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, upto, s);
            if (lane >= s) upto += o;
        }
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + upto > unit);
        if (past) {
            const int at = __ffs(past) - 1;
            b = first + at;
            tile = before + __shfl_sync(0xFFFFFFFFu, upto, at) - 1 - unit;
            return true;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return false;
}

// How the units (a tile under one KV head) are dealt to P CTAs. Whole rounds of P are not cut. The R < P units behind them would leave
// P - R multiprocessors idle for the time of a unit, so each is cut along its cached rows: into k = P / R large parts and, where
// P - kR CTAs are left over, a small one; a left-over CTA takes m = ceil(R / (P - kR)) small parts one after the other. Both take
// equally long when a large part has (m n + (m - 1) c) / (1 + k m) of the unit's n blocks; c: what a piece of work costs beside its
// blocks, in blocks. (64 units of 128 blocks on 148 multiprocessors: 176 us, 261 with every unit in two equal parts; 128
// units of 133 blocks: 404 us, 411 whole.)
constexpr int kPieceCost = 3, kLeastBlocks = 4, kLongBlocks = 32;
struct Deal {
    int whole, items;          // units that stay whole; pieces of work of all units
    int cut, k, m, parts;      // units that are cut, into at most `parts` parts
};
__device__ __forceinline__ Deal deal_of(int units, int ctas, bool split) {
    Deal d;
    d.whole = split ? units / ctas * ctas : units;
    d.cut = units - d.whole;
    d.k = d.parts = 1;
    d.m = 0;
    if (d.cut > 0) {
        d.k = ctas / d.cut;
        const int rest = ctas - d.k * d.cut;
        d.m = rest > 0 ? (d.cut + rest - 1) / rest : 0;
        d.parts = d.k + (rest > 0 ? 1 : 0);
    }
    d.items = d.whole + d.cut * d.parts;
    return d;
}
// Blocks of a large part of a cut unit of n blocks, and in `used` how many parts it has: 1 where cutting saves too little.
__device__ __forceinline__ int part_blocks(const Deal &d, int n, int &used) {
    // m < 2^8 and n < 2^24 for any count of multiprocessors below 2^8
    unsigned large = d.m > 0 ? ((unsigned)d.m * n + (d.m - 1) * kPieceCost + d.k * d.m) / (unsigned)(1 + d.k * d.m) : (unsigned)(n + d.k - 1) / (unsigned)d.k;
    if (large < kLeastBlocks) large = kLeastBlocks;
    used = 1;
    if (d.parts == 1 || large + kLeastBlocks >= (unsigned)n) return n;
    used = (int)((n + large - 1) / large);
    if (used > d.parts) used = d.parts;
    return (int)large;
}
// What the joining kernel has to know of a unit: its parts (1: it was not cut), sequence, first row and KV head.
struct __align__(16) CutUnit { int used, q_begin, rows, row0, head, slot, pad[2]; };

// Item `at` of the deal: its unit and part. Whole units first, then the large parts, then the small ones.
__device__ __forceinline__ int unit_of(const Deal &d, int at, int &part) {
    part = 0;
    if (at < d.whole) return at;
    part = (at - d.whole) / d.cut;
    return d.whole + (at - d.whole) % d.cut;
}

struct ManyArgs {
    AttentionArgs a;
    int few_rows;             // sequences of at most this many rows belong to the other kernel
    int tiles;                // upper bound of the tiles of all sequences
    CutUnit *cut_units;       // one for each CTA, with `split`
    int beside;               // the other kernel's launch follows and may begin as soon as this one has begun
    int split;                // whether units may be cut: the workspace is there, and cached rows enough for two parts
    uint64_t wait_limit_ns;
    int *status;
    int *next;                // two words, zero between launches: units handed out beyond the first of each CTA, CTAs that have ended
};
// One piece of work: 256 rows of one sequence against one part of its cached rows, under one KV head.
struct Work {
    int valid, b, head, used, tiles;
    int slot;                                 // of a part: its place in the workspace
    int row0, rows, q_begin, shift, q_len;    // shift: position of the sequence's first new token
    int begin, end;                           // cached rows of the part
    int pad;
    int blocks0, blocks1;                     // of each tile: the first tile's rows end earlier under a causal mask
    __device__ __forceinline__ int blocks(int i) const { return i == 0 ? blocks0 : blocks1; }
};

template <int DT, bool kEight, int DPAD>
__global__ void __launch_bounds__(kManyThreads, 1) attend_many_kernel(const __grid_constant__ ManyArgs args) {
    using Cfg = ManyCfg<DPAD, kEight>;
    constexpr int kBuffers = Cfg::kBuffers;
    const AttentionArgs &a = args.a;
    wait_for_predecessor();
    if (args.beside) let_next_begin();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t *base_ptr = smem_raw + (base - smem_addr(smem_raw));
    const uint32_t q_at = base, ring_at = base + 2 * Cfg::kTileBytes;
    uint8_t *raw_ptr = base_ptr + 2 * Cfg::kTileBytes + kBuffers * Cfg::kBufferBytes, *patches = raw_ptr + 2 * Cfg::kRawBytes, *tail = patches + Cfg::kPatchBytes;
    const uint32_t raw_at = ring_at + kBuffers * Cfg::kBufferBytes;
    Work *work = reinterpret_cast<Work *>(tail);                                  // two slots
    const uint32_t bars = smem_addr(tail + 2 * sizeof(Work));
    static_assert(sizeof(Work) % 8 == 0 && 2 * sizeof(Work) + 8 * (2 * 8 + 15) + 40 <= Cfg::kTailBytes, "tail of the shared memory");
    const uint32_t full0 = bars, empty0 = full0 + 8 * kBuffers, scores0 = empty0 + 8 * kBuffers, half0 = scores0 + 16, rest0 = half0 + 16,
                   done0 = rest0 + 16, q_full = done0 + 16, q_empty = q_full + 8, work_full0 = q_empty + 8, work_empty0 = work_full0 + 16,
                   want_next = work_empty0 + 16;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(tail + 2 * sizeof(Work) + 8 * (2 * kBuffers + 15));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dim = a.cache.dim, steps = dim >> 4;
    const uint64_t limit = args.wait_limit_ns;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kBuffers; ++i) { mbar_init(full0 + 8 * i, kLoaders); mbar_init(empty0 + 8 * i, 2); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(scores0 + 8 * i, 1); mbar_init(half0 + 8 * i, 4); mbar_init(rest0 + 8 * i, 4); mbar_init(done0 + 8 * i, 1);
            mbar_init(work_full0 + 8 * i, 1); mbar_init(work_empty0 + 8 * i, 14);
        }
        mbar_init(q_full, kLoaders); mbar_init(q_empty, 2); mbar_init(want_next, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr((const void *)tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Takes the next piece of work from its slot; the slot goes back at once. By whole warps. False: none left, or a wait ran out. While
    // the piece before (`w`) is at work nobody else hands anything on: that wait is allowed the time of its blocks as well.
    auto patience = [&](const Work &w) -> uint64_t { return limit + (uint64_t)max(w.blocks0, w.blocks1) * kBlockNs; };
    auto take_work = [&](int n, Work &w) -> bool {
        const int slot = n & 1;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(work_full0 + 8 * slot, (n >> 1) & 1, abort_flag, patience(w)))) return false;
        w = work[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(work_empty0 + 8 * slot);
        return w.valid != 0;
    };

    if (warp >= 8 && warp < 12) {
        // ===================== loader =====================
        give_registers<kLoaderRegs>();
        const int tid = threadIdx.x - 256;
        Work w = {};
        bool ok = true;
        int i = 0;                                                   // blocks of K and V so far, over all pieces of work
        for (int n = 0; ok && take_work(n, w); ++n) {
            // ---- queries, once the last product that reads the ones before has been done; rows behind the sequence are zeros
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(q_empty, (n & 1) ^ 1, abort_flag, limit));
            if (!ok) break;
            {
                constexpr int kChunks = DPAD / 8, kPass = kLoaders / kChunks;
                const int c = tid % kChunks, r0 = tid / kChunks, over = kPass % a.group, tokens = kPass / a.group;
                int token = (w.row0 + r0) / a.group, g = (w.row0 + r0) - token * a.group;
                const uint16_t *q = reinterpret_cast<const uint16_t *>(a.q.p) + (int64_t)w.q_begin * a.q.token_stride +
                                    (int64_t)w.head * a.group * a.q.head_stride + 8 * c;
                const uint32_t to = q_at + chunk_at(r0, c);
#pragma unroll 8
                for (int p = 0; p < 256; p += kPass) {
                    const bool there = w.row0 + r0 + p < w.rows;
                    if (8 * c < dim && p < 128 * w.tiles)
                        copy16(to + (p >> 7) * Cfg::kTileBytes + (p & 127) * 128, there ? q + token * a.q.token_stride + g * a.q.head_stride : q, there);
                    token += tokens; g += over;
                    if (g >= a.group) { g -= a.group; ++token; }
                }
                copy_commit();
            }
            bool q_pending = true;
            const int32_t *table = a.batch.table + (int64_t)w.b * a.batch.max_pages;
            const int blocks = w.blocks(w.tiles - 1);
            // lane i < 8 holds the page of cached rows 16 i .. 16 i + 15 of the block
            auto page_of = [&](int block) -> int {
                const int row = w.begin + block * kBlock + 16 * (lane & 7);
                return block < blocks && row < w.end ? table[row >> a.cache.page_shift] : 0;
            };
            int pages = page_of(0), next = 0, pending = -1;
            // 8-bit rows: thread = row of the block. It copies its codes to a place of its own two blocks ahead and turns them into
            // numbers when they are there, so that no thread waits for another; the row's exponent waits in a register. Through fp32
            // the way is two conversions and a product, which leaves the integer pipe to the softmax warps (with shifts and masks of
            // the codes instead a chunk on 16000 rows takes 439 us, so 414).
            int e0 = 0, e1 = 0, asked = pages, coming = 0;                // pages of the block asked for and of the one behind it
            auto ask = [&](int s) {
                if constexpr (kEight) {
                    if (s < 2 * blocks) {
                        const bool is_v = s & 1;
                        const int row = w.begin + (s >> 1) * kBlock + tid;
                        if (is_v) coming = page_of((s >> 1) + 1); else if (s > 0) asked = coming;
                        const int page = __shfl_sync(0xFFFFFFFFu, asked, tid >> 4);
                        const bool good = (uint32_t)page < (uint32_t)a.cache.pages, there = good && row < w.end;
                        const int64_t cell = ((int64_t)(good ? page : 0) * a.cache.kv_heads + w.head) * a.cache.page_size + (row & (a.cache.page_size - 1));
                        const uint8_t *from = (is_v ? a.cache.v : a.cache.k) + cell * dim;
                        const uint32_t to = raw_at + (s & 1) * Cfg::kRawBytes + tid * 16;
#pragma unroll
                        for (int c = 0; c < DPAD / 16; ++c)
                            if (16 * c < dim) copy16(to + c * 2048, from + 16 * c, there);
                        (is_v ? e1 : e0) = there ? (is_v ? a.cache.v_exp : a.cache.k_exp)[cell] : 0;
                        if (!good && !is_v) atomicOr(a.batch.status + kBatchWord, kBadPage);
                    }
                    copy_commit();
                }
            };
            ask(0);
            ask(1);
            const int nearly = blocks > 2 ? 2 * blocks - 4 : 0;           // two blocks before the end: in time for the next piece
            if (blocks == 0 && tid == 0) mbar_arrive(want_next);
            for (int s = 0; s < 2 * blocks; ++s, ++i) {
                const int buf = i % kBuffers;
                const bool is_v = s & 1;
                if (s == nearly && tid == 0) mbar_arrive(want_next);
                if (!kEight && !is_v) next = page_of((s >> 1) + 1);
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(empty0 + 8 * buf, ((i / kBuffers) & 1) ^ 1, abort_flag, limit));
                if (!ok) break;
                if constexpr (!kEight) {
                    const uint8_t *pool = is_v ? a.cache.v : a.cache.k;
                    const uint32_t dst = ring_at + buf * Cfg::kBufferBytes;
                    const int first = w.begin + (s >> 1) * kBlock;
                    constexpr int kChunks = DPAD / 8, kPass = kLoaders / kChunks;     // 128 threads bring kPass rows at a time, 8 or 16
                    const int c = tid % kChunks, r0 = tid / kChunks;
                    const uint32_t to = dst + chunk_at(r0, c);                         // kPass is a multiple of 8: the swizzle repeats
#pragma unroll
                    for (int g = 0; g < 8; ++g) {                                      // 16 rows lie in one page
                        const int page = __shfl_sync(0xFFFFFFFFu, pages, g);
                        const bool good = (uint32_t)page < (uint32_t)a.cache.pages;
                        const int64_t cell = ((int64_t)(good ? page : 0) * a.cache.kv_heads + w.head) * a.cache.page_size + ((first + 16 * g) & (a.cache.page_size - 1));
                        const uint8_t *from = pool + (cell + r0) * (2 * dim) + 16 * c;
#pragma unroll
                        for (int p = 0; p < 16; p += kPass) {
                            const bool there = good && first + 16 * g + r0 + p < w.end;
                            if (8 * c < dim) copy16(to + (16 * g + p) * 128, there ? from + p * (2 * dim) : pool, there);
                        }
                        if (!good && c == 0 && !is_v) atomicOr(a.batch.status + kBatchWord, kBadPage);
                    }
                    copy_commit();
                    copy_wait<1>();                                                    // all but the newest have landed
                    fence_async_shared();
                    if (q_pending) { mbar_arrive(q_full); q_pending = false; }
                    if (pending >= 0) mbar_arrive(full0 + 8 * pending);
                    pending = buf;
                } else {
                    // this thread's row of codes, asked for two blocks ago
                    if (q_pending) { copy_wait<2>(); fence_async_shared(); mbar_arrive(q_full); q_pending = false; }
                    copy_wait<1>();
                    const int e = s & 1 ? e1 : e0;
                    const uint4 *raw = reinterpret_cast<const uint4 *>(raw_ptr + (s & 1) * Cfg::kRawBytes) + tid;
                    uint8_t *out = base_ptr + 2 * Cfg::kTileBytes + buf * Cfg::kBufferBytes;
                    const float fs = row_scale(e);
#pragma unroll
                    for (int c = 0; c < DPAD / 16; ++c)
                        if (16 * c < dim) {
                            const uint4 x = raw[c * 128];
                            const uint32_t in[4] = {x.x, x.y, x.z, x.w};
                            uint32_t o[8];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float2 u = unpack2_e4m3(in[j]), v = unpack2_e4m3(in[j] >> 16);
                                o[2 * j] = pack2_rn<DT>(u.x * fs, u.y * fs);
                                o[2 * j + 1] = pack2_rn<DT>(v.x * fs, v.y * fs);
                            }
                            *reinterpret_cast<uint4 *>(out + chunk_at(tid, 2 * c)) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4 *>(out + chunk_at(tid, 2 * c + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    fence_async_shared();
                    mbar_arrive(full0 + 8 * buf);
                    ask(s + 2);
                }
                if (is_v) pages = next;
            }
            // the last block of this piece must not wait for the first of the next
            copy_wait<0>();
            fence_async_shared();
            if (ok && q_pending) mbar_arrive(q_full);
            if (ok && pending >= 0) mbar_arrive(full0 + 8 * pending);
        }
        copy_wait<0>();
    } else if (warp >= 12) {
        give_registers<kIssuerRegs>();
        if (warp == 12 || warp == 14) {
            // ===================== MMA issuer of one tile (one thread) =====================
            const int i = (warp - 12) >> 1;
            const uint32_t fmt = DT == MAGB200_BF16 ? 1u : 0u;
            const uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
            const uint32_t idesc_s = common | ((uint32_t)(kBlock >> 3) << 17);                       // N = 128 cached rows, both K-major
            const uint32_t idesc_o = common | (1u << 16) | ((uint32_t)(DPAD >> 3) << 17);            // N = head_dim, B MN-major
            const uint32_t s_at = tmem + 128u * i, o_at = tmem + Cfg::kOutCol + (uint32_t)(DPAD * i);
            const uint64_t qd = make_smem_desc(q_at + i * Cfg::kTileBytes, 16u, 1024u);
            const uint64_t kd0 = make_smem_desc(ring_at, 16u, 1024u), vd0 = make_smem_desc(ring_at, 128u * 128u, 1024u);
            Work w = {};
            bool ok = true;
            int fetched = 0, weighed = 0;                 // K and V blocks, weight tiles so far, over all pieces of work
            auto wait = [&](uint32_t bar, int phase) {
                ok = ok && mbar_wait(bar, (uint32_t)(phase & 1), abort_flag, limit);
                tcgen05_fence_after();
            };
            auto scores = [&](int buf) {
                const uint64_t kd = kd0 + (uint64_t)(buf * (Cfg::kBufferBytes >> 4));
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k)
                    if (k < steps) {
                        constexpr int kColumn = 128 * 128 >> 4;                                      // 64 elements further
                        mma_ss(s_at, qd + (uint64_t)((k >> 2) * kColumn + (k & 3) * 2), kd + (uint64_t)((k >> 2) * kColumn + (k & 3) * 2), idesc_s, k > 0);
                    }
                tcgen05_commit(scores0 + 8 * i);
            };
            // Each buffer is given back by both issuers. An issuer without products in a block (or, with one tile, in the whole
            // piece of work) still waits for every buffer and hands it back: a waiter that skipped a phase of a barrier would take
            // the phase before it for the one it waits for.
            auto release = [&](uint32_t bar, bool read) {
                if (read) tcgen05_commit(bar); else mbar_arrive(bar);
            };
            for (int n = 0; take_work(n, w); ++n) {
                const int blocks = w.blocks(w.tiles - 1), mine = i < w.tiles ? w.blocks(i) : 0;
                if (lane == 0) {
                    wait(q_full, n);
                    if (blocks > 0) {
                        wait(full0 + 8 * (fetched % kBuffers), fetched / kBuffers);
                        if (ok && mine > 0) scores(fetched % kBuffers);
                        if (ok) release(empty0 + 8 * (fetched % kBuffers), mine > 0);
                    }
                    if (ok && mine <= 1) release(q_empty, mine > 0);
                    for (int j = 0; ok && j < blocks; ++j, fetched += 2) {
                        const int v = fetched + 1, k = fetched + 2;
                        const uint64_t vd = vd0 + (uint64_t)((v % kBuffers) * (Cfg::kBufferBytes >> 4));
                        const bool more = j + 1 < blocks;
                        wait(full0 + 8 * (v % kBuffers), v / kBuffers);
                        if (j < mine) {
                            wait(half0 + 8 * i, weighed);
                            if (!ok) break;
#pragma unroll
                            for (int s = 0; s < 4; ++s) mma_ts(o_at, s_at + 8u * s, vd + 128u * s, idesc_o, j > 0 || s > 0);
                            if (more) wait(full0 + 8 * (k % kBuffers), k / kBuffers);       // ahead of the last wait before the next scores
                            wait(rest0 + 8 * i, weighed++);
                            if (!ok) break;
#pragma unroll
                            for (int s = 4; s < 8; ++s) mma_ts(o_at, s_at + 8u * s, vd + 128u * s, idesc_o, true);
                            if (j + 1 < mine) scores(k % kBuffers);
                            else tcgen05_commit(done0 + 8 * i);
                        } else if (more) {
                            wait(full0 + 8 * (k % kBuffers), k / kBuffers);
                        }
                        if (!ok) break;
                        release(empty0 + 8 * (v % kBuffers), j < mine);
                        if (more) {
                            release(empty0 + 8 * (k % kBuffers), j + 1 < mine);
                            if (j + 2 == mine) release(q_empty, true);
                        }
                    }
                }
                if (!__shfl_sync(0xFFFFFFFFu, (int)ok, 0)) break;
            }
        } else if (warp == 13) {
            // ===================== hands out the work =====================
            const Deal deal = deal_of(count_tiles(a, args.few_rows, args.tiles, lane) * a.cache.kv_heads, (int)gridDim.x, args.split != 0);
            int item = blockIdx.x;
            for (int n = 0;;) {
                Work w;
                memset(&w, 0, sizeof(w));
                bool found = item < deal.items;
                int part = 0, unit = 0;
                if (found) {
                    unit = unit_of(deal, item, part);
                    w.head = (int)(unit % a.cache.kv_heads);
                    int tile = 0, b = 0;
                    found = find_tile(a, args.few_rows, unit / a.cache.kv_heads, lane, b, tile);
                    w.b = b;
                    w.row0 = tile * kManyRows;
                }
                bool some = false;
                if (found) {
                    Tile t;
                    if (sequence_of(a, w.b, t) && w.row0 < t.rows) {
                        span_of(a, w.row0, kManyRows, t);
                        const int blocks = (int)((unsigned)(t.hi - t.lo + kBlock - 1) / kBlock);
                        const int per = unit < deal.whole ? (w.used = 1, blocks) : part_blocks(deal, blocks, w.used);
                        if (part < w.used) {
                            some = true;
                            const int begin = t.lo + part * per * kBlock, end = part + 1 < w.used ? begin + per * kBlock : t.hi;
                            w.slot = (unit - deal.whole) * deal.parts + part;
                            w.valid = 1;
                            w.tiles = w.row0 + 128 < t.rows ? 2 : 1;
                            w.rows = t.rows; w.q_begin = t.q_begin; w.q_len = t.q_len; w.shift = t.kv_len - t.q_len;
                            w.begin = begin; w.end = end > begin ? end : begin;
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                int to = end;
                                if (a.causal) {
                                    const int r = w.row0 + 128 * i + 127, token = (r < t.rows ? r : t.rows - 1) / a.group;
                                    if (w.shift + token + 1 < to) to = w.shift + token + 1;
                                }
                                (i == 0 ? w.blocks0 : w.blocks1) = to > begin ? (to - begin + kBlock - 1) / kBlock : 0;
                            }
                        }
                    }
                }
                if (some || !found) {
                    const int slot = n & 1;
                    if (!__all_sync(0xFFFFFFFFu, mbar_wait(work_empty0 + 8 * slot, ((n >> 1) & 1) ^ 1, abort_flag, limit))) break;
                    if (lane == 0) { work[slot] = w; mbar_arrive(work_full0 + 8 * slot); }
                    __syncwarp();
                    if (n == 0 && args.split) {                     // CTA i describes cut unit i, while its first piece of work runs
                        CutUnit c;
                        memset(&c, 0, sizeof(c));
                        const int cut = deal.whole + (int)blockIdx.x;
                        int b = 0, tile = 0;
                        Tile t;
                        if ((int)blockIdx.x < deal.cut && find_tile(a, args.few_rows, cut / a.cache.kv_heads, lane, b, tile) && sequence_of(a, b, t) &&
                            tile * kManyRows < t.rows) {
                            c.row0 = tile * kManyRows;
                            span_of(a, c.row0, kManyRows, t);
                            part_blocks(deal, (int)((unsigned)(t.hi - t.lo + kBlock - 1) / kBlock), c.used);
                            c.q_begin = t.q_begin; c.rows = t.rows; c.head = cut % a.cache.kv_heads; c.slot = (int)blockIdx.x * deal.parts;
                        }
                        if (lane == 0) args.cut_units[blockIdx.x] = c;
                    }
                    ++n;
                    if (!found) break;
                    // not before the loader nears the end of this piece: a CTA that took its next one earlier would keep it from one
                    // that has nothing to do (with up to two pieces taken ahead: prefill of 8 x 2048 tokens 429 us, so 407; a mixed batch 79, so 70)
                    if (!__all_sync(0xFFFFFFFFu, mbar_wait(want_next, (n - 1) & 1, abort_flag, patience(w)))) break;
                }
                int more = 0;
                if (lane == 0) more = atomicAdd(args.next, 1);
                item = (int)gridDim.x + __shfl_sync(0xFFFFFFFFu, more, 0);
            }
            // the last CTA to get here leaves the counters as the next launch expects them
            if (lane == 0) {
                __threadfence();
                if (atomicAdd(args.next + 1, 1) == (int)gridDim.x - 1) { args.next[0] = 0; args.next[1] = 0; }
            }
        }
    } else {
        // ===================== softmax =====================
        take_registers<kSoftmaxRegs>();
        const int i = warp >> 2, quarter = warp & 3;
        const float scale = a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2);
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + 128u * i, o_at = lanes + Cfg::kOutCol + (uint32_t)(DPAD * i);
        Work w = {};
        bool ok = true;
        int scored = 0, ended = 0;                                   // score tiles and pieces of work of this tile so far
        for (int n = 0; ok && take_work(n, w); ++n) {
            if (i >= w.tiles) continue;
            const int row = w.row0 + i * 128 + quarter * 32 + lane;
            const bool live = row < w.rows;
            const int token = (live ? row : w.rows - 1) / a.group, blocks = w.blocks(i);
            // cached rows seen_from .. seen_to - 1 are seen by this row, as offsets from the part's first
            int last = w.end, first = w.begin;
            if (a.causal) {
                if (w.shift + token + 1 < last) last = w.shift + token + 1;
                if (a.window > 0 && (int64_t)w.shift + token + 1 - a.window > first) first = (int)(w.shift + token + 1 - a.window);
            }
            const int seen_to = last > w.begin ? last - w.begin : 0, seen_from = first - w.begin;
            float ref = -CUDART_INF_F, sum = 0.0f;
            for (int j = 0; j < blocks; ++j, ++scored) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(scores0 + 8 * i, scored & 1, abort_flag, limit));
                if (!ok) break;
                tcgen05_fence_after();
                const int from = seen_from - j * kBlock, to = seen_to - j * kBlock;       // of this block's 128 columns
                const bool whole = __all_sync(0xFFFFFFFFu, from <= 0 && to >= kBlock);
                float x[kBlock];
                tmem_load_row<128>(s_at, x);
                // the maximum is taken before scaling: a negative scale moves its sign to the scores, a scale of zero makes them
                // zeros (infinities and NaN stay what the product with the scale makes of them)
                if (a.scale_log2 <= 0.0f) {
                    const float f = a.scale_log2 < 0.0f ? -1.0f : 0.0f;
#pragma unroll
                    for (int c = 0; c < kBlock; ++c) x[c] *= f;
                }
                if (!whole) mask_columns<kBlock>(x, from, to);
                // The first half's weights are made with the reference as it stands while the row's maximum is found; in the rare
                // block that moves the reference they are made again from the scores, which are still in TMEM.
                auto exponentials = [&](int c0, float minus) {
#pragma unroll
                    for (int c = c0; c < c0 + 64; c += 2) {
                        fma2(x[c], x[c + 1], scale, minus);
                        x[c] = exp2_fast(x[c]);
                        x[c + 1] = exp2_fast(x[c + 1]);
                    }
                };
                auto minus_ref = [&]() { return ref == -CUDART_INF_F ? 0.0f : fmaf(-ref, scale, kLift<DT>); };
                float top;
                {
                    float tops[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int c = 4; c < 124; c += 8) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) tops[y] = max3(tops[y], x[c + y], x[c + 4 + y]);
                    }
#pragma unroll
                    for (int y = 0; y < 4; ++y) tops[y] = fmaxf(tops[y], x[124 + y]);
                    top = max3(tops[0], tops[1], fmaxf(tops[2], tops[3]));
                }
                exponentials(0, minus_ref());
                // a row that has seen nothing yet has no reference; its weights are exp2(-inf) = 0 against any
                const bool move = top > -CUDART_INF_F && (ref == -CUDART_INF_F || (top - ref) * scale > kMoveAt);
                if (__any_sync(0xFFFFFFFFu, move)) {
                    const float factor = move ? (ref == -CUDART_INF_F ? 0.0f : exp2_fast((ref - top) * scale)) : 1.0f;
                    if (move) ref = top;
                    sum *= factor;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < DPAD; c += 16) {
                            uint32_t r[16];
                            tmem_load_16(o_at + c, r);
#pragma unroll
                            for (int y = 0; y < 16; ++y) r[y] = __float_as_uint(__uint_as_float(r[y]) * factor);
                            tmem_st_32x16(o_at + c, r);
                        }
                    }
                    tmem_load_row<64>(s_at, x);
                    if (a.scale_log2 <= 0.0f) {
                        const float f = a.scale_log2 < 0.0f ? -1.0f : 0.0f;
#pragma unroll
                        for (int c = 0; c < 64; ++c) x[c] *= f;
                    }
                    if (!whole) mask_columns<64>(x, from, to);
                    exponentials(0, minus_ref());
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half == 1) exponentials(64, minus_ref());
#pragma unroll
                    for (int c = 64 * half; c < 64 * half + 64; c += 32) {
                        uint32_t p[16];
#pragma unroll
                        for (int y = 0; y < 32; y += 2) p[y >> 1] = pack2_rn<DT>(x[c + y], x[c + y + 1]);
                        tmem_st_32x16(s_at + (c >> 1), p);      // over columns whose scores are in registers
                    }
                    tmem_st_wait();
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive((half == 0 ? half0 : rest0) + 8 * i);   // the product with half of the block can start
                }
                float part[4] = {x[0], x[1], x[2], x[3]};       // beside the product
#pragma unroll
                for (int c = 4; c < kBlock; c += 4) { add2(part[0], part[1], x[c], x[c + 1]); add2(part[2], part[3], x[c + 2], x[c + 3]); }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
            }
            if (ok && blocks > 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(done0 + 8 * i, (ended++) & 1, abort_flag, limit));
            if (!ok) break;
            tcgen05_fence_after();
            const int64_t heads = a.q.heads, out_token = (int64_t)w.q_begin + token, qh = (int64_t)w.head * a.group + (row - token * a.group);
            const float inv = w.used > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
            if (w.used > 1) {
                // a warp's rows side by side: [maximum and sum of 32 rows][four elements of 32 rows]..., 512 bytes with every store
                float4 *part = reinterpret_cast<float4 *>(a.partial + ((int64_t)w.slot * kManyRows + i * 128 + quarter * 32) * (dim + 4)) + lane;
#pragma unroll 1
                for (int c = 0; c < dim; c += 16) {
                    uint32_t r[16];
                    if (blocks > 0) {
                        tmem_load_16(o_at + c, r);
                    } else {                                                       // the tile's rows end before this part
#pragma unroll
                        for (int y = 0; y < 16; ++y) r[y] = 0u;
                    }
#pragma unroll
                    for (int y = 0; y < 16; y += 4)
                        part[32 * (1 + (c + y) / 4)] = make_float4(__uint_as_float(r[y]), __uint_as_float(r[y + 1]), __uint_as_float(r[y + 2]), __uint_as_float(r[y + 3]));
                }
                part[0] = make_float4(ref == -CUDART_INF_F ? ref : ref * scale, sum, 0.0f, 0.0f);
            } else {
                // 64 columns at a time through the warp's patch of shared memory (a row's 16-byte chunks XOR-swizzled by the row),
                // from which eight lanes write 128 bytes of one row: a lane that wrote its own row would touch 32 lines with
                // every store (5.2 k clocks of the 16 k that a piece of work took beside its blocks)
                uint8_t *patch = patches + warp * 4096;
                const uint64_t dst = reinterpret_cast<uint64_t>(reinterpret_cast<uint16_t *>(a.out.p) + out_token * a.out.token_stride + qh * a.out.head_stride);
                const uint32_t alive = __ballot_sync(0xFFFFFFFFu, live);
#pragma unroll 1
                for (int c0 = 0; c0 < dim; c0 += 64) {
                    float r[64];
                    if (blocks > 0) {
                        tmem_load_row<64>(o_at + c0, r);
                    } else {
#pragma unroll
                        for (int y = 0; y < 64; ++y) r[y] = 0.0f;
                    }
                    __syncwarp();                                                  // the patch has been read
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        uint4 o;
                        o.x = pack2_rn<DT>(r[8 * y + 0] * inv, r[8 * y + 1] * inv);
                        o.y = pack2_rn<DT>(r[8 * y + 2] * inv, r[8 * y + 3] * inv);
                        o.z = pack2_rn<DT>(r[8 * y + 4] * inv, r[8 * y + 5] * inv);
                        o.w = pack2_rn<DT>(r[8 * y + 6] * inv, r[8 * y + 7] * inv);
                        *reinterpret_cast<uint4 *>(patch + lane * 128 + ((y ^ (lane & 7)) << 4)) = o;
                    }
                    __syncwarp();
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        const int rr = 4 * y + (lane >> 3), c = lane & 7;
                        const uint64_t to = __shfl_sync(0xFFFFFFFFu, dst, rr);
                        const uint4 o = *reinterpret_cast<const uint4 *>(patch + rr * 128 + ((c ^ (rr & 7)) << 4));
                        if ((alive >> rr & 1u) && c0 + 8 * c < dim) *reinterpret_cast<uint4 *>(to + 2 * (c0 + 8 * c)) = o;
                    }
                }
            }
            const float m = ref == -CUDART_INF_F ? ref : ref * scale;
            if (live && w.used == 1 && a.lse) a.lse[out_token * heads + qh] = sum == 0.0f ? -CUDART_INF_F : (m + log2f(sum * pow2f(-(int)kLift<DT>))) * kLn2;
        }
    }
    // ---- end: everyone meets, then the TMEM goes back. After a wait that ran out, products in flight get time to land first.
    __syncwarp();
    if (*abort_flag) {
        if (threadIdx.x == 0) atomicExch(args.status, kTimeoutStatus);
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) { }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---- joining the parts of cut units -----------------------------------------------------------------------------------------
// A CTA has 32 rows of a cut unit, one to a lane, and each of its warps eight elements; parts are taken in their order, so that
// results are the same from call to call.
constexpr int kJoinThreads = 512;
template <int DT> __global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttentionArgs a, const CutUnit *units) {
    wait_for_predecessor();
    const CutUnit c = units[blockIdx.x];
    const int used = c.used;
    if (used <= 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = a.cache.dim, row = c.row0 + blockIdx.y * 32 + lane;
    if (8 * warp >= dim) return;
    const int64_t step = (int64_t)kManyRows * (dim + 4) / 4;
    const float4 *part = reinterpret_cast<const float4 *>(a.partial + ((int64_t)c.slot * kManyRows + blockIdx.y * 32) * (dim + 4)) + lane;
    float m = -CUDART_INF_F, l = 0.0f;
#pragma unroll 8
    for (int i = 0; i < used; ++i) m = fmaxf(m, part[i * step].x);
    const float ref = m == -CUDART_INF_F ? 0.0f : m;
    float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
#pragma unroll 4
    for (int i = 0; i < used; ++i) {
        const float4 *p = part + i * step;
        const float4 s = p[0], x = p[32 * (1 + 2 * warp)], y = p[32 * (2 + 2 * warp)];
        const float w = exp2_fast(s.x - ref);
        l = fmaf(w, s.y, l);
        u.x = fmaf(w, x.x, u.x); u.y = fmaf(w, x.y, u.y); u.z = fmaf(w, x.z, u.z); u.w = fmaf(w, x.w, u.w);
        v.x = fmaf(w, y.x, v.x); v.y = fmaf(w, y.y, v.y); v.z = fmaf(w, y.z, v.z); v.w = fmaf(w, y.w, v.w);
    }
    if (row >= c.rows) return;
    const int token = row / a.group;
    const int64_t to = (int64_t)c.q_begin + token, qh = (int64_t)c.head * a.group + (row - token * a.group);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *dst = reinterpret_cast<uint16_t *>(a.out.p) + to * a.out.token_stride + qh * a.out.head_stride + 8 * warp;
    *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2_rn<DT>(u.x * inv, u.y * inv), pack2_rn<DT>(u.z * inv, u.w * inv),
                                                 pack2_rn<DT>(v.x * inv, v.y * inv), pack2_rn<DT>(v.z * inv, v.w * inv));
    if (a.lse && warp == 0) a.lse[to * a.q.heads + qh] = l == 0.0f ? -CUDART_INF_F : (m + log2f(l * pow2f(-(int)kLift<DT>))) * kLn2;   // sums and outputs of parts are scaled alike
}

template <int DT, bool kEight, int DPAD> int launch(const ManyArgs &m, int ctas, cudaStream_t st, bool early) {
    constexpr int kSmem = ManyCfg<DPAD, kEight>::kSmem;
    if (int rc = opt_in_shared<attend_many_kernel<DT, kEight, DPAD>, kSmem>()) return rc;
    return launch_kernel(attend_many_kernel<DT, kEight, DPAD>, dim3((unsigned)ctas), kManyThreads, kSmem, st, early, m);
}
template <int DT> int launch_all(const ManyArgs &m, int ctas, cudaStream_t st, bool early) {
    if (m.a.cache.bits == 8) return m.a.cache.dim <= 64 ? launch<DT, true, 64>(m, ctas, st, early) : launch<DT, true, 128>(m, ctas, st, early);
    return m.a.cache.dim <= 64 ? launch<DT, false, 64>(m, ctas, st, early) : launch<DT, false, 128>(m, ctas, st, early);
}
ManyArgs many_args(const AttentionArgs &a, const AttentionPlan &p) {
    ManyArgs m;
    m.a = a; m.few_rows = p.few_rows;
    // A unit that is cut has more than 2 kLeastBlocks blocks; fewer than 2 parts for every CTA have to be held. From two rounds on the
    // queue alone keeps the multiprocessors busy, and the second kernel costs what cutting the rest saves (a prefill of 8 x 2048 tokens:
    // 409 us, 417 with its last 136 units in parts).
    // The bound on the units counts one for every sequence, also those of the streaming kernel. Where it reaches two rounds, but the
    // rows behind those of single tokens fill less than half a round and a unit may be long, units are cut as well (64 tokens of
    // 64 heads on 100000 rows beside 60 single tokens, 16 units: 1750 us whole, 370 cut). Short or many units are not worth it (16 single
    // tokens beside 8 prompts of 500 with a window of 1024, 180 units: 58 us whole, 65 cut; behind 4000 rows: 118 and 128).
    const size_t parts = (size_t)a.ctas * 2 * kManyRows * (a.cache.dim + 4) * sizeof(float);
    const int64_t least_units = (a.batch.tokens * a.group - (int64_t)a.batch.batch * p.few_rows) / kManyRows * a.cache.kv_heads;
    const bool less_than_two_rounds = p.many_tiles * a.cache.kv_heads < 2 * a.ctas;
    const bool few_long_units = 2 * least_units < a.ctas && p.many_keys > kLongBlocks * kBlock;
    m.split = (less_than_two_rounds || few_long_units) && p.many_keys > 2 * kLeastBlocks * kBlock && parts + a.ctas * sizeof(CutUnit) <= a.partial_bytes;
    m.cut_units = reinterpret_cast<CutUnit *>(reinterpret_cast<char *>(a.partial) + parts);
    m.tiles = (int)p.many_tiles;
    m.beside = p.few_ctas > 0;
    m.wait_limit_ns = get_wait_limit_ns();
    m.status = a.batch.status;
    m.next = a.batch.status + kWorkWord;
    return m;
}

}  // namespace

int launch_attend_many(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st, bool early) {
    const ManyArgs m = many_args(a, p);
    const int64_t units = p.many_tiles * a.cache.kv_heads;
    const int ctas = m.split || units > a.ctas ? a.ctas : (int)units;
    return a.cache.dtype == MAGB200_BF16 ? launch_all<MAGB200_BF16>(m, ctas, st, early) : launch_all<MAGB200_F16>(m, ctas, st, early);
}
int launch_join_many(const AttentionArgs &a, const AttentionPlan &p, cudaStream_t st) {
    const ManyArgs m = many_args(a, p);
    if (!m.split) return MAGB200_OK;
    const dim3 grid((unsigned)a.ctas, kManyRows / 32);
    const CutUnit *units = m.cut_units;
    return a.cache.dtype == MAGB200_BF16 ? launch_kernel(join_kernel<MAGB200_BF16>, grid, kJoinThreads, 0, st, true, a, units)
                                         : launch_kernel(join_kernel<MAGB200_F16>, grid, kJoinThreads, 0, st, true, a, units);
}

}  // namespace magb200
