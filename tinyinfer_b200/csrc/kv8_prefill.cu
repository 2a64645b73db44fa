// mp_kv8_attention_prefill: causal attention of packed chunks of rows over the 8-bit
// paged cache, on tcgen05 (sm_100a).
//
// A work item is (block of rows of one sequence, kv head): rows x query heads of the group
// fill two 128-vector tiles (vector v of a tile: row v / group, head v % group), and its
// context is a run of 128-token K/V tiles. All items' tiles, in order, are dealt out in
// runs of equal cost to one CTA per SM (an item's queries and outputs count too), so a long
// context with few rows is shared like many short ones; the device plans this itself from
// row_offsets and starts.
//
// Calls with few rows go to kv8_decode.cu's kernel (launch_prefill below).
//
// Roles of a CTA (three more warps idle):
//  * warps 8-11 widen K and V codes to FP16 tiles in shared memory (exact; K token-major,
//    V token-major too: the tensor core reads it transposed), with their blocks' scales. The codes
//    come by cp.async: loaded into registers a tile ahead, they waited for one another in the
//    little L1 that the tiles leave (8 x 1024 rows of 32 / 8 heads x 128 BF16: 452 us, now 383);
//  * one lane of warp 12 issues the products: S = Q K^T into tensor memory, O = P V with
//    P from tensor memory;
//  * warps 0-3 and 4-7 own one tile each, a thread per vector: running softmax of S's
//    row, weights written over S in place, O's rows added up. (Two threads per vector,
//    with half of the tokens and dims each, measured 13-15 % slower: they have to tell each
//    other their largest scores, and a thread then has too few registers.)
// S has kBuffers places (3 x 128 columns beside two O of 64, 2 beside two O of 128), used in
// turn by both tiles: with three, a tile's next S is ready before its threads ask for it.
//
// Outputs: FP32 ones are added up in registers, tile by tile; BF16 ones stay in tensor
// memory over kChainTiles of an item's tiles, and chains are added up in the workspace.
//
// FP32 precision: the query is two FP16 halves (each row scaled by a power of two towards
// FP16's top), so S is two products per useful one; the weights, with V's scales folded
// in, are two halves as well. BF16 inputs and outputs take one of each. The tensor core
// cuts its sums (measured: 9e-8 of the sum per product of 16), so O starts anew with
// every 128 tokens and is added up in FP32 registers, and the small halves' products go
// first.
//
// Bound by the softmax's chain of instructions: of the 6100 cycles that 256 vectors x 128 tokens
// take in FP32 at head_dim 64 (16 x 512 rows of 9 / 3 heads at position 3584: 247 us), a thread
// spends 900 on the maximum, 2900 on the weights, 640 on O and 700 waiting; an item's start and
// end cost 700 more per tile. exp2 alone would take 2050, the products 2050 (3100 measured: P V is
// 64 wide). At head_dim 128 BF16 (8 x 1024 rows of 32 / 8 heads at position 1000: 382 us, 531
// TFLOP/s) it is 8000 cycles: 3600 of softmax, 2800 of waiting for S, whose place is free only after
// the tile's own P V, 1500 of items' starts and ends.
#include <algorithm>

#include "kv8.cuh"
#include "umma.cuh"

namespace mpb {
namespace kv8 {
namespace {

constexpr int kWidenWarp = 8, kProductWarp = 12, kThreads = 512;
constexpr int kM = 128;       // vectors of a tile
constexpr int kN = 128;       // tokens of a K/V tile
// Scale rows in flight. Row j + 4 is written after P V of tile j + 1 completed (its V slot
// was needed for tile j + 3), so every thread has read row j by then.
constexpr int kScaleSlots = 4;
// Costs that runs are dealt out by: a K/V tile for both tiles of vectors, an item's start and end (8 and
// 12 within 1 % of 10), and kAloneCost, a K/V tile for one tile of vectors: items of one take 0.73 to
// 0.75 of the time of two at head_dim 128, 0.81 (FP32) and 0.93 (BF16) at 64.
constexpr int kPairCost = 4, kSetup = 10;
constexpr int kGroupTokens = 16;  // tokens that share a block's scales at least
constexpr int kGroups = kN / kGroupTokens;
// A weight times V scale of `unit` is 2^8 in FP16, and may grow to 2^15 before the reference
// score and the unit move (kRoom): a move costs a third of a tile's softmax, and with room for
// 2^2 some row of a warp asked for one in most tiles. FP16's smallest half step, 2^-25, is
// 2^-33 of the largest.
constexpr int kTopLog = 8;
// K/V tiles of one chain of sums in tensor memory (BF16 outputs): 2048 products, each of which may cut 2^-23
// of the sum, 2.4e-4 in all, an eighth of BF16's half step. (An uncut item of 2^20 tokens came out 5e-3
// small in one chain.)
constexpr int kChainTiles = 256;
constexpr float kRoom = 7.f;

template <class T, int D>
struct Shape {
    static constexpr int kHalves = sizeof(T) == 4 ? 2 : 1;              // FP16 halves of q and of the weights
    static constexpr int kTileBytes = kM * D * 2;                       // one FP16 tile
    static constexpr bool kAdd = kHalves == 2;                          // O starts anew with every tile
    static constexpr int kStages = kHalves == 2 && D == 128 ? 1 : 2;    // K (and V) tiles in shared memory
    static constexpr int kQ = 0;                                        // [2 tiles][halves]
    static constexpr int kK = kQ + 2 * kHalves * kTileBytes;
    static constexpr int kV = kK + kStages * kTileBytes;
    static constexpr int kRing = D == 64 ? 3 : 1;                       // tiles of codes in flight, as they are
    static constexpr int kRaw = kV + kStages * kTileBytes;              // [ring][K, V][words of a thread][128 threads]
    static constexpr int kRawScales = kRaw + kRing * 2 * kN * D;        // [ring][groups] K, V
    static constexpr int kScales = kRawScales + kRing * kGroups * 8;    // [slots][groups] K, V, log2 V, 1 / V
    static constexpr int kBars = kScales + kScaleSlots * kGroups * 16;
    static constexpr int kPlan = kQ;                                    // before the queries come
    static constexpr int kSmem = kBars + 32 * 8;
    static constexpr int kAlloc = kSmem + 1024;                         // alignment slack
    static constexpr int kBuffers = D == 64 ? 3 : 2;                    // places of S
    // registers a thread of each role: together those of the launch, 512 x 128
    static constexpr int kSoftmaxRegs = 184, kWidenRegs = 72;
    static constexpr int kProductRegs = 512 - 2 * kSoftmaxRegs - kWidenRegs;
    static constexpr int kAloneCost = D == 128 ? 3 : 4;
    static constexpr uint32_t kTmemCols = 512;                          // S: kBuffers x 128, O: 2 x D
};
static_assert(Shape<float, 128>::kAlloc <= 232448 && Shape<__nv_bfloat16, 128>::kAlloc <= 232448);

// Descriptor of an MN-major operand tile: rows of 128 bytes (64 elements of the MN
// dimension), 8-row groups of 1024 bytes along K, 64-element blocks kTileRows rows apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t tile, uint32_t block_bytes) {
    uint64_t d = (tile >> 4) & 0x3FFFull;
    d |= uint64_t(block_bytes >> 4) << 16;
    d |= uint64_t(1024 >> 4) << 32;
    d |= uint64_t(1) << 46;
    d |= uint64_t(2) << 61;
    return d;
}

// D (TMEM) (+)= A (TMEM) . B, one K step of 16 FP16 elements.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// Columns of this warp's TMEM lanes, waited for: a register of a load in flight must not be
// moved, and the compiler does not know that it is.
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15"
        "}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24,"
        "%25, %26, %27, %28, %29, %30, %31"
        "}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31,"
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47,"
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63"
        "}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
          "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
          "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
          "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
          "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
        : "r"(taddr));
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Packed pairs of FP32 (two 32-bit registers side by side).
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 unpair(Pair p) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) {
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
    return p;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b) {
    Pair p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
// split_pair of a packed pair
__device__ __forceinline__ void split_packed(Pair p, Pair minus_one, uint32_t& hi, uint32_t& lo) {
    const float2 v = unpair(p);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(h);
    const float2 rest = unpair(fma_pair(pair(f.x, f.y), minus_one, p));
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Registers a thread of this warpgroup from here on; the launch gives 128.
template <int N>
__device__ __forceinline__ void set_registers() {
    if constexpr (N > 128) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
    }
}

__device__ __forceinline__ void copy_row16(uint32_t to, const void* from, bool live) {  // zeros where not live
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ void copy_scales(uint32_t to, const float* from, bool live) {  // zeros where not live
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(live ? 8 : 0) : "memory");
}
// All but the youngest N groups of this thread's copies are done.
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The values of a 16-byte word.
__device__ __forceinline__ void widen_word(uint4 w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void widen_word(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
}

// One item's tiles k0 .. k1 - 1 (of `tiles`), and what it covers.
struct Segment {
    int seq, row0, rows, position, head, k0, k1, tiles, cost;
    int64_t first;  // device-wide index of the item's first unit of cost (its tiles follow kSetup units)
};

// The blocks of rows of all sequences in order, and a run of their tiles.
template <int kAloneCost>
struct RunCursor {
    const AttentionParams* p;
    int block_rows;  // rows of a full item
    int seq, block, head, k;  // k: unit of the item
    int64_t at;               // device-wide index of the next unit
    int left;
    int begin, start, rows;   // of sequence `seq`

    static __device__ __forceinline__ int tiles_of(int start, int rows, int block, int block_rows) {
        return (start + min((block + 1) * block_rows, rows) + kN - 1) / kN;
    }
    static __device__ __forceinline__ int cost_of(int rows, int block, int block_rows) {
        return 2 * (rows - block * block_rows) <= block_rows ? kAloneCost : kPairCost;
    }
    static __device__ __forceinline__ int units_of(int start, int rows, int block, int block_rows) {
        return kSetup + cost_of(rows, block, block_rows) * tiles_of(start, rows, block, block_rows);
    }
    // The next segment; false when the run is done.
    __device__ __forceinline__ bool next(Segment& s) {
        do
            if (!advance(s)) return false;
        while (s.k0 >= s.k1);  // no tile of the item begins in the run
        return true;
    }
    __device__ __forceinline__ bool advance(Segment& s) {
        if (left <= 0) return false;
        while (block * block_rows >= rows) {
            block = 0, head = 0, k = 0;
            rows = sequence_rows(*p, ++seq, begin, start);
        }
        s.seq = seq, s.head = head;
        s.row0 = begin + block * block_rows;
        s.rows = min(block_rows, rows - block * block_rows);
        s.position = start + block * block_rows;
        const int tiles = tiles_of(start, rows, block, block_rows), cost = cost_of(rows, block, block_rows);
        const int end = min(kSetup + cost * tiles, k + left);
        s.tiles = tiles, s.cost = cost;
        // the tiles whose first unit is in the run
        s.k0 = max(k - kSetup + cost - 1, 0) / cost, s.k1 = max(end - kSetup + cost - 1, 0) / cost;
        s.first = at - k;
        left -= end - k, at += end - k;
        k = 0;
        if (++head == p->cache.kv_heads) head = 0, ++block;
        return true;
    }
};

// kLong: BF16 outputs of contexts that may pass one chain (launch_prefill)
template <class T, int F, int D, bool kLong>
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const AttentionParams p) {
    using S = Shape<T, D>;
    using Cursor = RunCursor<S::kAloneCost>;
    constexpr int kHalves = S::kHalves, kStages = S::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float4* scales = reinterpret_cast<float4*>(sm + S::kScales);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::kBars);
    uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;
    uint64_t *q_full = bars + 8, *p_full = bars + 10, *o_full = bars + 12, *joined = bars + 14, *q_free = bars + 16;  // per tile
    uint64_t *s_full = bars + 18, *scales_full = bars + 21;  // per place of S; per row of scales
    uint64_t* done = bars + 25;                              // a segment's products
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 26);
    int* failed = reinterpret_cast<int*>(bars + 27);
    uint64_t* drained = bars + 29;                           // products in flight after a wait that expired
    int* last = reinterpret_cast<int*>(bars + 28);  // [2] whether this CTA joins the parts, per tile
    int64_t* units_before = reinterpret_cast<int64_t*>(sm + S::kPlan);       // [kThreads + 1]
    int64_t* sums = units_before + kThreads + 1;                         // [32], [32]
    int* blocks_before = reinterpret_cast<int*>(sums + 64);                  // [kThreads + 1]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == kProductWarp) tmem_alloc(tmem_holder, S::kTmemCols);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, 4), mbar_init(v_full + i, 4);
            mbar_init(k_empty + i, 1), mbar_init(v_empty + i, 1);
            mbar_init(q_full + i, 4), mbar_init(p_full + i, 4), mbar_init(o_full + i, 1);
            mbar_init(joined + i, 4), mbar_init(q_free + i, 4);
        }
        for (int i = 0; i < S::kBuffers; ++i) mbar_init(s_full + i, 1);
        for (int i = 0; i < kScaleSlots; ++i) mbar_init(scales_full + i, 1);
        mbar_init(done, 1), mbar_init(drained, 1);
        *failed = 0;
        fence_barrier_init();
    }
    pdl_enter();

    // ---- plan: blocks of rows of each thread's sequences, then units of each thread's blocks
    const int group = p.heads / p.cache.kv_heads, tile_rows = kM / group, block_rows = 2 * tile_rows;
    const int share = (p.count + kThreads - 1) / kThreads;
    auto scan = [&](int64_t mine, int64_t* partial) {  // exclusive sum over the threads before
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) partial[warp] = upto;
        __syncthreads();
        int64_t x = lane < warp ? partial[lane] : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x + upto - mine;
    };
    int begin, start;
    {
        int mine = 0, falls = 0;
        for (int i = tid * share; i < min((tid + 1) * share, p.count); ++i) {
            mine += (sequence_rows(p, i, begin, start) + block_rows - 1) / block_rows;
            falls |= p.row_offsets[i + 1] < begin;
        }
        const int before = int(scan(mine, sums));
        blocks_before[tid] = before;
        if (tid == kThreads - 1) blocks_before[kThreads] = before + mine;
        // offsets that fall may rise again and name rows many times over, up to 2^44 blocks of them, past
        // the indexes below: such a call is left out (reported above)
        if (__syncthreads_or(falls) && tid == kThreads - 1) blocks_before[kThreads] = 0;
        __syncthreads();
    }
    const int blocks = blocks_before[kThreads], each = (blocks + kThreads - 1) / kThreads;
    // sequence and block of the flattened block index `f` (< blocks)
    auto locate = [&](int f, int& seq, int& block) {
        int t = 0;
#pragma unroll
        for (int o = kThreads / 2; o; o >>= 1)
            if (blocks_before[t + o] <= f) t += o;
        block = f - blocks_before[t];
        for (seq = t * share;; ++seq) {
            const int n = (sequence_rows(p, seq, begin, start) + block_rows - 1) / block_rows;
            if (block < n) return;
            block -= n;
        }
    };
    {
        int64_t mine = 0;
        if (tid * each < blocks) {
            int seq, block;
            locate(tid * each, seq, block);
            int rows = sequence_rows(p, seq, begin, start);
            for (int i = 0; i < min(each, blocks - tid * each); ++i, ++block) {
                while (block * block_rows >= rows) block = 0, rows = sequence_rows(p, ++seq, begin, start);
                mine += Cursor::units_of(start, rows, block, block_rows);
            }
        }
        const int64_t before = scan(mine, sums + 32);
        units_before[tid] = before;
        if (tid == kThreads - 1) units_before[kThreads] = before + mine;
        __syncthreads();
    }
    const int heads = p.cache.kv_heads;
    const int64_t total = units_before[kThreads] * heads;
    // every run holds a tile's first unit wherever it lies in an item
    const int ctas = int(min(total / kPairCost, int64_t(gridDim.x)));
    const int64_t base = ctas ? (total >> 32 ? total / ctas : int64_t(uint32_t(total) / uint32_t(ctas))) : 0;
    const int extra = int(total - base * ctas);
    auto cta_of = [&](int64_t unit) {
        const int64_t split = extra * (base + 1);
        return int(unit < split ? unit / (base + 1) : extra + (unit - split) / base);
    };
    Cursor cursor{&p, block_rows};
    if (base >= kMostUnits) raise_error(p.error, kErrBounds);
    cursor.left = int(blockIdx.x) < ctas && base < kMostUnits ? int(base) + (int(blockIdx.x) < extra) : 0;
    if (cursor.left) {
        cursor.at = blockIdx.x * base + min(int(blockIdx.x), extra);
        int t = 0;
#pragma unroll
        for (int o = kThreads / 2; o; o >>= 1)
            if (units_before[t + o] * heads <= cursor.at) t += o;
        locate(t * each, cursor.seq, cursor.block);
        int64_t in = cursor.at - units_before[t] * heads;
        cursor.rows = sequence_rows(p, cursor.seq, cursor.begin, cursor.start);
        for (;; ++cursor.block) {
            while (cursor.block * block_rows >= cursor.rows)
                cursor.block = 0, cursor.rows = sequence_rows(p, ++cursor.seq, cursor.begin, cursor.start);
            const int n = Cursor::units_of(cursor.start, cursor.rows, cursor.block, block_rows);
            if (in < int64_t(n) * heads) {
                cursor.head = int(in) / n, cursor.k = int(in) % n;
                break;
            }
            in -= int64_t(n) * heads;
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_holder;
    // tiles of a segment that tile w's rows see: none if it has no rows
    auto tiles_for = [&](const Segment& s, int w) {
        const int rows = min(s.rows, (w + 1) * tile_rows);
        return rows <= w * tile_rows ? 0 : max(0, min(s.k1, (s.position + rows + kN - 1) / kN) - s.k0);
    };
    // Bounded wait of one thread, or of a whole warp (whose lanes then agree). After a wait
    // that expired every role leaves its loops at its next wait.
    auto wait_one = [&](uint64_t* bar, uint32_t parity) {
        for (int i = 0; i < 64; ++i)  // before the clock is read, which takes longer than most waits
            if (mbar_try_wait(bar, parity)) return true;
        const uint64_t start = global_ns(), limit = p.stall_ns ? p.stall_ns : kWaitNanoseconds;
        while (!*reinterpret_cast<volatile int*>(failed) && global_ns() - start < limit)
            if (mbar_try_wait(bar, parity)) return true;
        *reinterpret_cast<volatile int*>(failed) = 1;
        raise_error(p.error, kErrTimeout);
        return false;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_one(bar, parity)) != 0; };

    if (warp < kWidenWarp) {
        // ================================================================ softmax, a thread per vector
        set_registers<S::kSoftmaxRegs>();
        const int w = warp >> 2, v = tid & (kM - 1);
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t o_at = tmem + S::kBuffers * kN + w * D + lanes;
        unsigned char* q_tile = sm + S::kQ + w * kHalves * S::kTileBytes;
        const float sign = p.scale < 0.f ? -1.f : 1.f;  // the sign goes to q: scores' factors stay positive
        uint32_t o_phase = 0, join_phase = 0, free_phase = 1;
        int slot = 0, used = 0;  // K/V tiles and S places that earlier segments took
        Segment seg;
        bool ok = true;
        auto arrive = [&](uint64_t* bar) {  // of the warp
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        while (ok && cursor.next(seg)) {
            const int n0 = tiles_for(seg, 0), n1 = tiles_for(seg, 1), tiles = w ? n1 : n0, most = seg.k1 - seg.k0;
            const int row = w * tile_rows + v / group;
            const bool live = v < tile_rows * group && row < seg.rows;
            const int position = seg.position + row;
            float o[D], m = -INFINITY, l = 0.f, k_factor = 0.f;
            int unit_log = -110;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] = 0.f;
            // The segment before is done, and the tile's other warps have left its query buffer. (A tile
            // with fewer tokens, or none, would else run ahead, and S's places and the scales are waited for
            // by the parity of their phase: one phase ahead passes for the one before.)
            if (!(ok = wait(q_free + w, free_phase)) || !(ok = wait(done, free_phase))) break;
            free_phase ^= 1;
            if (tiles) {
                // ---- query rows as FP16 halves, K-major with the 128-byte swizzle. A warp brings its rows, as they
                // are, to where their halves go, then a lane takes its row to registers and writes the halves back
                constexpr int kWords = D * int(sizeof(T)) / 16, kEach = 16 / int(sizeof(T)), kCols = D / 64;
                const int r0 = v & ~31;
                const uint64_t from = reinterpret_cast<uint64_t>(
                    live ? static_cast<const T*>(p.q) + int64_t(seg.row0 + row) * p.q_stride + (seg.head * group + v % group) * D
                         : nullptr);
                auto place = [&](int r, int word) {  // of a row's raw 16-byte word
                    const int piece = word / 8;      // 128 bytes: a column block of a half
                    return piece / kCols * S::kTileBytes + piece % kCols * (kM * 128) + int(sw128_offset(r, word % 8));
                };
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const int x = i * 32 + lane, r = x / kWords, word = x % kWords;
                    const uint64_t at = __shfl_sync(0xffffffffu, from, r);
                    copy_row16(smem_u32(q_tile) + place(r0 + r, word),
                               at ? reinterpret_cast<const char*>(at) + word * 16 : static_cast<const char*>(p.q), at != 0);
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                __syncwarp();
                uint4 raw[kWords];
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    raw[i] = *reinterpret_cast<const uint4*>(q_tile + place(v, i));
                    float x[kEach];
                    widen_word(raw[i], x);
#pragma unroll
                    for (int c = 0; c < kEach; ++c) amax = fmaxf(amax, fabsf(x[c]));
                }
                float factor, inverse;
                row_factor(amax, factor, inverse);
                k_factor = inverse * (p.scale * sign) * kLog2e;
                factor *= sign;
                __syncwarp();  // every lane has read its words
#pragma unroll
                for (int i = 0; i < D; i += 8) {
                    uint32_t hi[4], lo[4];
                    float x[8];
                    if constexpr (kEach == 8) {
                        widen_word(raw[i / 8], x);
                    } else {
                        widen_word(raw[i / 4], *reinterpret_cast<float(*)[4]>(x));
                        widen_word(raw[i / 4 + 1], *reinterpret_cast<float(*)[4]>(x + 4));
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) split_pair(x[2 * c] * factor, x[2 * c + 1] * factor, hi[c], lo[c]);
                    unsigned char* to = q_tile + i / 64 * (kM * 128) + sw128_offset(v, i % 64 / 8);
                    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (kHalves == 2)
                        *reinterpret_cast<uint4*>(to + S::kTileBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_proxy_async_shared();
            }
            arrive(q_full + w);
            // O's row of this thread, times `by`
            auto add_outputs = [&](float by) {
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    float x[32];
                    tmem_load(o_at + i, x);
                    const Pair bb = pair(by, by);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 s = unpair(fma_pair(pair(x[j], x[j + 1]), bb, pair(o[i + j], o[i + j + 1])));
                        o[i + j] = s.x, o[i + j + 1] = s.y;
                    }
                }
            };
            // a part of the item in the workspace, vectors side by side. Slot 0 of a CTA: the item began
            // earlier, slot 1: it begins here. A segment's own slot is free until its end: chains go there
            constexpr int64_t kPart = int64_t(kM) * (D + 2);
            float* parts = reinterpret_cast<float*>(static_cast<unsigned char*>(p.workspace) + kCounterBytes);
            auto part = [&](int cta, int which) { return parts + ((int64_t(cta) * 2 + which) * 2 + w) * kPart; };
            [[maybe_unused]] float chain_m = -INFINITY;  // reference score of the finished chains
            // BF16: a chain of outputs, in plain units, out of tensor memory
            [[maybe_unused]] auto end_chain = [&](bool first) {
                const float unit = pow2(unit_log - kTopLog), decay = chain_m == m ? 1.f : ex2(chain_m - m);
                float* mine = part(blockIdx.x, seg.k0 == 0) + v * 4;
#pragma unroll 1
                for (int i = 0; i < D; i += 16) {
                    float x[16];
                    tmem_load(o_at + i, x);
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        float4* at = reinterpret_cast<float4*>(mine + (i + c) * kM);
                        float4 sum = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
                        sum.x = fmaf(x[c], unit, sum.x * decay), sum.y = fmaf(x[c + 1], unit, sum.y * decay);
                        sum.z = fmaf(x[c + 2], unit, sum.z * decay), sum.w = fmaf(x[c + 3], unit, sum.w * decay);
                        *at = sum;
                    }
                }
                chain_m = m;
            };
            for (int j = 0; j < tiles; ++j) {
                // S places in order: j = 0 of both tiles, j = 1, ..., each as far as it goes
                const int place = used + (w ? min(j + 1, n0) + j : j + min(j, n1));
                if (!(ok = wait(s_full + place % S::kBuffers, (place / S::kBuffers) & 1))) break;
                tmem_fence_after();
                const uint32_t s_at = tmem + place % S::kBuffers * kN + lanes;
                bool behind = j > 0;  // O of the tile before is still to come
                auto wait_outputs = [&] {
                    if (behind) {
                        ok = wait(o_full + w, o_phase);
                        o_phase ^= 1;
                        behind = false;
                        tmem_fence_after();
                    }
                    return ok;
                };
                const int sl = (slot + j) % kScaleSlots;
                if (!(ok = wait(scales_full + sl, ((slot + j) / kScaleSlots) & 1))) break;
                const float4* scale = scales + sl * kGroups;
                // tokens of the tile that the row sees (padding vectors are zero queries: all, so that they
                // bring no masks into their warp)
                const int visible = live ? min(max(position + 1 - (seg.k0 + j) * kN, 0), kN) : kN;
                const bool cut = __any_sync(0xffffffffu, visible < kN);
                // f(x, g) for every group of 16 scores, `at_once` of them per load
                auto each_group = [&](auto at_once, auto f) {
                    constexpr int kAtOnce = decltype(at_once)::value;
#pragma unroll 1
                    for (int g = 0; g < kGroups; g += kAtOnce) {
                        float x[16 * kAtOnce];
                        tmem_load(s_at + g * 16, x);
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) f(*reinterpret_cast<float(*)[16]>(x + 16 * i), g + i);
                    }
                };
                using One = std::integral_constant<int, 1>;
                float moved = 1.f;  // factor of the outputs so far
                // the tile's weights; kCut: some row of the warp does not see all of its tokens
                auto weigh = [&](auto is_cut) {
                    constexpr bool kCut = decltype(is_cut)::value;
                    // (64 scores at once: BF16, head_dim 64, 16 x 512 rows at position 3584 take 185 us, 198 with
                    // 32; in the other shapes too few registers are left: FP32 259 and 249, head_dim 128 405 and 383)
                    using Some = std::integral_constant<int, kCut || (S::kAdd && D == 128) ? 1 : !S::kAdd && D == 64 ? 4 : 2>;
                    auto largest_of = [&](float (&x)[16], int g) {  // scaled
                        if constexpr (kCut) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[i] = g * 16 + i < visible ? x[i] : -INFINITY;
                        }
                        float big = fmaxf(x[0], x[1]);
#pragma unroll
                        for (int i = 2; i < 16; i += 2) big = max3(big, x[i], x[i + 1]);
                        return kCut && g * 16 >= visible ? -INFINITY : big * (k_factor * scale[g].x);
                    };
                    float top = -INFINITY, reach = -INFINITY;  // largest score, and log2 of weight times V scale plus m
                    each_group(Some{}, [&](float (&x)[16], int g) {
                        const float t = largest_of(x, g);
                        top = fmaxf(top, t);
                        reach = fmaxf(reach, t + scale[g].z);
                    });
                    const bool high = reach - m > float(unit_log) + kRoom || top > m + 20.f;
                    if (__any_sync(0xffffffffu, high)) {
                        if (high) {
                            const float m_new = fmaxf(m, top);
                            const float decay = m == -INFINITY ? 0.f : ex2(m - m_new);
                            // the largest so far, in whole powers of two; within the exponents of floats
                            const float most = fmaxf(m == -INFINITY ? -110.f : float(unit_log) + (m - m_new), reach - m_new);
                            const int next = int(floorf(fminf(fmaxf(most, -110.f), 126.f)));
                            moved = m == -INFINITY ? 0.f : ex2(m - m_new + float(unit_log - next));
                            l *= decay;
                            m = m_new, unit_log = next;
                        }
                        if constexpr (S::kAdd) {
#pragma unroll
                            for (int d = 0; d < D; ++d) o[d] *= moved;
                        } else if (j) {
                            if (!wait_outputs()) return;
#pragma unroll 1
                            for (int i = 0; i < D; i += 16) {
                                float x[16];
                                tmem_load(o_at + i, x);
#pragma unroll
                                for (int c = 0; c < 16; ++c) x[c] *= moved;
                                tmem_store8(o_at + i, *reinterpret_cast<uint32_t(*)[8]>(x));
                                tmem_store8(o_at + i + 8, *reinterpret_cast<uint32_t(*)[8]>(x + 8));
                            }
                        }
                    }
                    // weight * V scale = 2^(score - m + log2 scale - log2 unit + 8). A scale below unit * 2^-60
                    // counts as that: its weights (up to 2^20 * 2^-52) are zero in FP16 either way, but l needs them
                    const float base_m = m == -INFINITY ? 0.f : m, shift = float(kTopLog - unit_log);
                    const float unit = pow2(unit_log);
                    [[maybe_unused]] const Pair minus_one = pair(-1.f, -1.f);
                    const float least = fmaxf(unit * 8.6736174e-19f, 1.17549435e-38f);
                    float tile_l = 0.f;  // the tile's weights first: fewer additions to a long sum
                    each_group(Some{}, [&](float (&x)[16], int g) {
                        const float4 sc = scale[g];
                        const bool small = sc.y < least;
                        const float f = k_factor * sc.x;
                        const float c = (small ? float(kTopLog - 60) : sc.z + shift) - base_m;
                        const float back = small ? 4503599627370496.f : sc.w * (unit * (1.f / (1 << kTopLog)));
                        const Pair ff = pair(f, f), cc = pair(c, c);
                        Pair sum = pair(0.f, 0.f);
                        uint32_t hi[8];
                        [[maybe_unused]] uint32_t lo[8];
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const float2 t = unpair(fma_pair(pair(x[i], x[i + 1]), ff, cc));
                            float p0 = ex2(t.x), p1 = ex2(t.y);
                            if constexpr (kCut) {
                                p0 = g * 16 + i < visible ? p0 : 0.f;
                                p1 = g * 16 + i + 1 < visible ? p1 : 0.f;
                            }
                            const Pair pp = pair(p0, p1);
                            sum = add_pair(sum, pp);
                            if constexpr (kHalves == 2) {
                                split_packed(pp, minus_one, hi[i / 2], lo[i / 2]);
                            } else {
                                const __half2 packed = __floats2half2_rn(p0, p1);
                                hi[i / 2] = *reinterpret_cast<const uint32_t*>(&packed);
                            }
                        }
                        const float2 both = unpair(sum);
                        tile_l = fmaf(both.x + both.y, kCut && g * 16 >= visible ? 0.f : back, tile_l);
                        // over the scores just read: 16 columns hold 8 of high halves, 8 of low
                        tmem_store8(s_at + g * 16, hi);
                        if constexpr (kHalves == 2) tmem_store8(s_at + g * 16 + 8, lo);
                    });
                    l += tile_l;
                };
                if (cut) {
                    weigh(std::true_type{});
                } else {
                    weigh(std::false_type{});
                }
                // the last tile's O, its weights relative to the reference before this tile
                if (!ok || !wait_outputs()) break;
                if (S::kAdd && j) add_outputs(moved);
                tmem_wait_store();
                if (kLong && j && j % kChainTiles == 0) end_chain(j == kChainTiles);
                tmem_fence_before();
                arrive(p_full + w);
            }
            if (ok && tiles && (ok = wait(o_full + w, o_phase))) {
                o_phase ^= 1;
                tmem_fence_after();
                add_outputs(1.f);
                tmem_fence_before();
            }
            used += n0 + n1;
            slot += most;
            if (!ok) break;
            const float u = pow2(unit_log - kTopLog);
            if (kLong && tiles > kChainTiles) {
                const float* mine = part(blockIdx.x, seg.k0 == 0) + v * 4;
                const float by = (chain_m == m ? 1.f : ex2(chain_m - m)) / u;
#pragma unroll
                for (int d = 0; d < D; d += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(mine + d * kM);
                    o[d] = fmaf(x.x, by, o[d]), o[d + 1] = fmaf(x.y, by, o[d + 1]);
                    o[d + 2] = fmaf(x.z, by, o[d + 2]), o[d + 3] = fmaf(x.w, by, o[d + 3]);
                }
            }
            // rows out through this tile's query buffer (its products are done): the warp's 32 rows,
            // 16-byte words XOR-ed by the row against bank conflicts, then word by word
            auto write_rows = [&](float r) {
                constexpr int kWords = D * int(sizeof(T)) / 16, kEach = 16 / int(sizeof(T));
                unsigned char* stage = q_tile + (warp & 3) * 32 * (kWords * 16);
                const uint64_t to_row = reinterpret_cast<uint64_t>(
                    live ? static_cast<T*>(p.out) + int64_t(seg.row0 + row) * p.out_stride + (seg.head * group + v % group) * D
                         : nullptr);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    T* to = reinterpret_cast<T*>(stage + lane * (kWords * 16) + (i ^ (lane & 7)) * 16);
#pragma unroll
                    for (int c = 0; c < kEach; c += 4)
                        store4(to + c, o[i * kEach + c] * r, o[i * kEach + c + 1] * r, o[i * kEach + c + 2] * r, o[i * kEach + c + 3] * r);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const int x = i * 32 + lane, from = x / kWords, word = x % kWords;
                    const uint64_t at = __shfl_sync(0xffffffffu, to_row, from);
                    if (at)
                        reinterpret_cast<uint4*>(at)[word] =
                            *reinterpret_cast<const uint4*>(stage + from * (kWords * 16) + (word ^ (from & 7)) * 16);
                }
            };
            if (seg.k0 == 0 && seg.k1 == seg.tiles) {
                if (tiles) write_rows(l == 0.f ? 0.f : u / l);
                arrive(q_free + w);
                continue;
            }
            // ---- a part of the item: to the workspace; the last CTA to arrive joins them
            unsigned* counters = static_cast<unsigned*>(p.workspace);
            auto state = [&](int cta, int which) { return parts + (((int64_t(cta) * 2 + which) * 2 + w) * kPart + D * kM + v * 2); };
            {
                float* mine = part(blockIdx.x, seg.k0 == 0);
#pragma unroll
                for (int d = 0; d < D; d += 4)
                    *reinterpret_cast<float4*>(mine + d * kM + v * 4) =
                        make_float4(o[d] * u, o[d + 1] * u, o[d + 2] * u, o[d + 3] * u);
                *reinterpret_cast<float2*>(state(blockIdx.x, seg.k0 == 0)) = make_float2(m, l);
            }
            __threadfence();
            auto meet = [&] {  // the tile's four warps
                arrive(joined + w);
                ok = wait(joined + w, join_phase);
                join_phase ^= 1;
                return ok;
            };
            if (!meet()) break;
            const int c0 = cta_of(seg.first + kSetup), n = cta_of(seg.first + kSetup + seg.cost * (seg.tiles - 1)) - c0 + 1;
            if (v == 0) {
                const bool mine_last = atomicAdd(counters + 2 * c0 + w, 1u) == unsigned(n - 1);
                if (mine_last) counters[2 * c0 + w] = 0;
                last[w] = mine_last;
                __threadfence();
            }
            if (!meet()) break;
            if (*reinterpret_cast<volatile int*>(last + w)) {
                m = -INFINITY, l = 0.f;
#pragma unroll
                for (int d = 0; d < D; ++d) o[d] = 0.f;
                for (int i = 0; i < n; ++i) {
                    const float* from = part(c0 + i, i == 0);
                    const float2 ml = __ldcg(reinterpret_cast<const float2*>(state(c0 + i, i == 0)));
                    const float big = fmaxf(m, ml.x);
                    const float a = m == big ? 1.f : ex2(m - big), b = ml.x == big ? 1.f : ex2(ml.x - big);
                    l = l * a + ml.y * b;
                    m = big;
#pragma unroll
                    for (int d = 0; d < D; d += 4) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(from + d * kM + v * 4));
                        o[d] = fmaf(o[d], a, x.x * b), o[d + 1] = fmaf(o[d + 1], a, x.y * b);
                        o[d + 2] = fmaf(o[d + 2], a, x.z * b), o[d + 3] = fmaf(o[d + 3], a, x.w * b);
                    }
                }
                write_rows(l == 0.f ? 0.f : 1.f / l);
            }
            if (!meet()) break;  // `last` may be written again
            arrive(q_free + w);
        }
    } else if (warp < kProductWarp) {
        // ================================================================ codes -> FP16 tiles
        set_registers<S::kWidenRegs>();
        const int t = tid & 127, bt = p.cache.block_tokens;
        constexpr int kWords = kN * D / 16 / 128;  // 16-byte words of a thread per tile
        constexpr int kChunks = D / 16;            // words of a token
        const int first_token = t / kChunks, chunk = t % kChunks, in_page = bt / kGroupTokens;
        const int own = first_token % kGroupTokens * D + chunk * 16;
        const uint32_t raw = smem_u32(sm + S::kRaw) + t * 16, raw_scales = smem_u32(sm + S::kRawScales);
        // the word's 16 FP16 values in a tile: two 16-byte chunks of the token's row
        const int to0 = (chunk / 4) * (kN * 128) + int(sw128_offset(first_token, 2 * (chunk % 4)));
        const int to1 = (chunk / 4) * (kN * 128) + int(sw128_offset(first_token, 2 * (chunk % 4) + 1));
        int slot = 0;
        Segment seg;
        bool ok = true;
        while (ok && cursor.next(seg)) {
            const int32_t* table = p.tables + int64_t(seg.seq) * p.table_stride;
            const int len = seg.position + seg.rows;
            // Codes and scales are copied kRing tiles ahead; a thread copies what it widens itself. The
            // blocks of four tiles at a time are found by the lanes, 8 pieces of 16 tokens each: their
            // K rows' offsets (V's are one block of rows on); table entries are read four tiles earlier.
            const int first = slot - seg.k0;
            int64_t offset = 0;
            int block = 0, entry, rest;
            auto peek = [&](int k) {
                const int piece = k * kGroups + lane, page = piece / in_page;
                entry = 0, rest = piece - page * in_page;
                if (piece < seg.k1 * kGroups && piece * kGroupTokens < len) entry = page < p.table_stride ? table[page] : -1;
            };
            auto copy = [&](int k, int part) {
                if (k < seg.k1) {
                    const int place = (first + k) % S::kRing, in = (k - seg.k0) % 4 * kGroups, left = len - k * kN;
                    if (part == 0) {
                        if (in == 0) {
                            block = checked_id(p.cache, entry, p.error);
                            offset = tile_offset(p.cache, block, seg.head, 0, D) + rest * (kGroupTokens * D);
                            peek(k + 4);
                        }
                        const int from = __shfl_sync(0xffffffffu, block, in + lane % kGroups);
                        if (t < kGroups)
                            copy_scales(raw_scales + (place * kGroups + t) * 8, p.cache.scales + from * p.cache.scale_stride + 2 * seg.head,
                                        t * kGroupTokens < left);
                    }
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        const int64_t at = __shfl_sync(0xffffffffu, offset, in + first_token / kGroupTokens + i * (kN / kWords) / kGroupTokens);
                        const bool live = first_token + i * (kN / kWords) < left;
                        copy_row16(raw + ((place * 2 + part) * kWords + i) * 2048, p.cache.pages + (live ? at + part * bt * D + own : 0), live);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");  // one per tile and part, empty ones included
            };
            peek(seg.k0);
            for (int k = seg.k0; k < seg.k0 + S::kRing; ++k) copy(k, 0), copy(k, 1);
            for (int k = seg.k0; ok && k < seg.k1; ++k, ++slot) {
                const int stage = slot % kStages;
                const uint32_t parity = ((slot / kStages) & 1) ^ 1;
                const int place = slot % S::kRing;
                wait_copies<2 * S::kRing - 1>();
                if (t < kGroups) {
                    const float2 scale = *reinterpret_cast<const float2*>(sm + S::kRawScales + (place * kGroups + t) * 8);
                    scales[slot % kScaleSlots * kGroups + t] =
                        make_float4(scale.x, scale.y, __log2f(scale.y), scale.y == 0.f ? 0.f : 1.f / scale.y);
                }
                __syncwarp();
                if (t == 0) mbar_arrive(scales_full + slot % kScaleSlots);
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    if (part && p.stall_ns) ok = false;
                    if (!ok || !(ok = wait((part ? v_empty : k_empty) + stage, parity))) break;
                    if (part) wait_copies<2 * S::kRing - 1>();
                    unsigned char* tile = sm + (part ? S::kV : S::kK) + stage * S::kTileBytes;
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        const uint4 c = *reinterpret_cast<const uint4*>(sm + S::kRaw + ((place * 2 + part) * kWords + i) * 2048 + t * 16);
                        uint32_t h[8];
                        widen4<F>(c.x, h[0], h[1]);
                        widen4<F>(c.y, h[2], h[3]);
                        widen4<F>(c.z, h[4], h[5]);
                        widen4<F>(c.w, h[6], h[7]);
                        unsigned char* to = tile + i * (kN / kWords) * 128;  // whole groups of 8 rows on: same swizzle
                        *reinterpret_cast<uint4*>(to + to0) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4*>(to + to1) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive((part ? v_full : k_full) + stage);
                    copy(k + S::kRing, part);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ================================================================ products
        set_registers<S::kProductRegs>();
        if (warp == kProductWarp) {
            // the warp runs in step and one elected lane issues: the descriptors stay in uniform registers
            constexpr uint32_t kIdescS = umma_idesc_f16<kM, kN>();
            constexpr uint32_t kIdescO = umma_idesc_f16<kM, D>() | (1u << 16);  // B is MN-major
            // descriptors' low bits are addresses / 16: adding moves them
            const uint64_t q_desc = smem_desc(sm + S::kQ), k_desc = smem_desc(sm + S::kK);
            const uint64_t v_desc = mn_desc(smem_u32(sm + S::kV), kN * 128);
            int slot = 0, used = 0;  // as in the softmax
            uint32_t q_phase = 0, p_phase = 0;  // p_phase: one bit per tile
            Segment seg;
            bool ok = true;
            while (ok && cursor.next(seg)) {
                const int most = __shfl_sync(0xffffffffu, seg.k1 - seg.k0, 0);
                const int n0 = __shfl_sync(0xffffffffu, tiles_for(seg, 0), 0), n1 = __shfl_sync(0xffffffffu, tiles_for(seg, 1), 0);
                // (tile, K/V tile) pairs in order: `s` the next S, `o` the next O, kBuffers behind it
                struct Next {
                    int w, j;
                    __device__ __forceinline__ void skip(int n0, int n1, int most) {
                        while (j < most && j >= (w ? n1 : n0)) step();
                    }
                    __device__ __forceinline__ void step() { w ^= 1, j += w == 0; }
                };
                Next s{0, 0}, o{0, 0};
                s.skip(n0, n1, most), o.skip(n0, n1, most);
                if (!(ok = wait(q_full, q_phase) && wait(q_full + 1, q_phase))) break;
                q_phase ^= 1;
                for (int i = 0; ok && i < n0 + n1 + S::kBuffers; ++i) {
                    if (i >= S::kBuffers) {
                        const int stage = (slot + o.j) % kStages, place = (used + i - S::kBuffers) % S::kBuffers;
                        ok = wait(p_full + o.w, (p_phase >> o.w) & 1) && wait(v_full + stage, ((slot + o.j) / kStages) & 1);
                        if (!ok) break;
                        p_phase ^= 1u << o.w;
                        tmem_fence_after();
                        const uint32_t s_at = tmem + place * kN, o_at = tmem + S::kBuffers * kN + o.w * D;
                        const uint64_t vd = v_desc + uint64_t(stage * (S::kTileBytes >> 4));
                        const bool keep = !S::kAdd && (kLong ? o.j % kChainTiles : o.j) != 0, leave = o.w || o.j >= n1;  // leave: V's last use
                        if (elect()) {
#pragma unroll
                            for (int half = kHalves - 1; half >= 0; --half)
#pragma unroll
                                for (int c = 0; c < kN / 16; ++c)
                                    mma_f16_ts(o_at, s_at + c * 16 + half * 8, vd + uint64_t(c * (2048 >> 4)), kIdescO,
                                               half != kHalves - 1 || c != 0 || keep);
                            mma_commit(o_full + o.w);
                            if (leave) mma_commit(v_empty + stage);
                        }
                        __syncwarp();
                        o.step(), o.skip(n0, n1, most);
                    }
                    if (i < n0 + n1) {
                        const int stage = (slot + s.j) % kStages, place = (used + i) % S::kBuffers;
                        ok = wait(k_full + stage, ((slot + s.j) / kStages) & 1);
                        if (!ok) break;
                        tmem_fence_after();
                        const uint32_t s_at = tmem + place * kN;
                        const uint64_t kd = k_desc + uint64_t(stage * (S::kTileBytes >> 4));
                        const uint64_t qd = q_desc + uint64_t(s.w * kHalves * (S::kTileBytes >> 4));
                        const bool leave = s.w || s.j >= n1;
                        if (elect()) {
#pragma unroll
                            for (int half = kHalves - 1; half >= 0; --half)
#pragma unroll
                                for (int c = 0; c < D / 16; ++c)
                                    mma_f16(s_at, qd + uint64_t(half * (S::kTileBytes >> 4) + (c / 4) * (kM * 128 >> 4) + c % 4 * 2),
                                            kd + uint64_t((c / 4) * (kN * 128 >> 4) + c % 4 * 2), kIdescS,
                                            half != kHalves - 1 || c != 0);
                            mma_commit(s_full + place);
                            if (leave) mma_commit(k_empty + stage);
                        }
                        __syncwarp();
                        s.step(), s.skip(n0, n1, most);
                    }
                }
                if (!ok) break;
                if (elect()) mma_commit(done);
                __syncwarp();
                slot += most, used += n0 + n1;
            }
        }
        __syncwarp();
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == kProductWarp) {
        if (*failed) {  // the roles left in mid-work: products may still be using the tiles and tensor memory
            if (elect()) mma_commit(drained);
            __syncwarp();
            mbar_wait_bounded(drained, 0);
        }
        tmem_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

}  // namespace

size_t prefill_workspace(int group, int head_dim) {
    return std::max(decode_workspace(group, head_dim), kCounterBytes + size_t(kCtas) * 4 * kM * (head_dim + 2) * 4);
}

cudaError_t launch_prefill(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    // Few rows go one by one, as decode's do, while there is an SM for each (row, kv head, 8 query
    // heads): their tokens are read once per row, but no tile of vectors has to be filled. 9 / 3
    // heads, FP32, beside the tiles: 37 rows 7.6 us against 13.4 (at position 500 11.6 / 19.8);
    // 49 rows 8.0 / 14.8, at 2000 17.0 / 30.0, at 16000 63 / 67.9. Twice as many would
    // still gain a little on short contexts (98 rows 14.6 / 15.0, at 2000 27.2 / 31.6), and lose
    // on long ones, where the time is the tokens that an SM passes over.
    if (int64_t(p.rows) * p.cache.kv_heads * ((p.heads / p.cache.kv_heads + 7) / 8) <= kPackedItems)
        return launch_packed(p, type, format, head_dim, stream);
    return dispatch(type, format, head_dim, [&](auto t, auto f, auto d) {
        using T = decltype(t);
        constexpr int kFormat = decltype(f)::value, kDim = decltype(d)::value;
        using S = Shape<T, kDim>;
        auto launch = [&](auto kernel) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kAlloc);
            if (e != cudaSuccess) return e;
            return launch_pdl(kernel, dim3(kCtas), dim3(kThreads), S::kAlloc, stream, p);
        };
        // Ending chains takes registers from the loop over tiles (BF16: 16 x 512 rows of 9 / 3 heads x 64 at position
        // 3584 200 us, 185 without; 8 x 1024 of 32 / 8 heads x 128 at 1000 387, 380): tables that cannot hold a
        // context longer than a chain go without.
        if constexpr (!S::kAdd)
            if (int64_t(p.table_stride) * p.cache.block_tokens > int64_t(kChainTiles) * kN)
                return launch(prefill_kernel<T, kFormat, kDim, true>);
        return launch(prefill_kernel<T, kFormat, kDim, false>);
    });
}

}  // namespace kv8
}  // namespace mpb
