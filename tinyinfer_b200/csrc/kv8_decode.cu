// mp_kv8_attention_decode: one query row per sequence over the 8-bit paged cache (sm_100a);
// and the rows of small mp_kv8_attention_prefill calls (kPacked).
//
// A token costs 2 head_dim bytes per kv head and 4 head_dim flops per query head. The work
// is cut into units of 32 tokens of one (row, kv head, up to 8 query heads) item; all items'
// units, in order, are dealt out in equal runs to one CTA per SM and its warps, however
// long the sequences are, or a CTA takes an item whole. The lengths are device memory,
// so every CTA adds them up itself (a block scan) and finds where its warps' runs begin.
//
// A warp works on its own: cp.async fills its ring of 1 to 3 units in shared memory (rows
// swizzled against bank conflicts), the warp-level tensor ops of kv8_warp.cuh empty it, and no
// two warps wait for one another before the end. At head_dim 64 16 warps keep up to 192 KB in
// flight per SM; FP32 at 128 has 8 warps with two units or more; BF16 at 128 12 warps, whose
// partials leave room for one unit each from 3 query heads per kv head on: nothing is then in
// flight while such a warp computes, the others cover for it. (The copy engine's tiles, issued by
// a lane, cost the warp more instructions than 16-byte copies by all lanes: 74 us against 52 for
// 256 rows of 2048 tokens.)
//
// Bound by instructions at head_dim 64: about 480 a unit on a scheduler with 4 warps, where the
// ring without arithmetic takes 40 us for 256 x 2048 tokens of 9 / 3 heads; with it 55 us in FP32
// (3.7 TB/s), 50 in BF16. At 128, 64 x 4096 tokens of 32 / 8 heads take 102 us in FP32 (5.3 TB/s),
// nearer to HBM, and 110 in BF16 (4.9 TB/s), with the one-unit rings.
//
// An item that ends in a later run leaves partials (max, sum, outputs): a CTA's warps join theirs
// through shared memory, CTAs through the workspace: the last CTA to arrive on the counter of
// the CTA in which the item began joins them in CTA order (deterministic) and clears it.
#include "kv8_warp.cuh"

namespace mpb {
namespace kv8 {
namespace {

constexpr int kSmemBytes = 227 * 1024;
// Units per warp before another CTA takes part (1 is no faster; with 4, one row of 32768 tokens took
// 20.7 us instead of 17.9).
constexpr int kMinUnits = 2;
// Units per warp that a CTA may take beyond its equal share to have an item whole, if there is a CTA for
// each: no CTA then waits for another. Against runs: one row of 333 tokens 8.9 us (12.2), 3 x 1000 11.8
// (12.8), 49 x 2000 16.6 (21.7), 64 x 4096 of 16 / 2 heads x 128 40.0 (43.8). With 2, 24 x 3000 takes
// 20.8 us, 19.6 with 4; with 6, 16 rows at position 4000 take 22.4, 20.1 with 4.
constexpr int kWholeUnits = 4;

template <class T, int D>
__host__ __device__ constexpr int warps_of() {
    return D == 64 ? 16 : sizeof(T) == 2 ? 12 : 8;  // 128, 168 and 255 registers a thread
}

struct Record {  // a partial of one warp, or none (units 0)
    int64_t first;  // device-wide index of the item's first unit
    int row, item, units;
    int begins, ends;  // it holds the item's first / last unit
};

// Shared memory of a CTA; `heads` = partial rows (query heads of an item, up to 8).
struct Layout {
    int partials, records, meta, misc, total, stages;
};
__host__ __device__ constexpr Layout layout_of(int warps, int heads, int head_dim) {
    Layout l{};
    const int stage = 2 * kUnit * head_dim;  // [tile][K, V][16 tokens][head_dim]
    const int partial = heads * (head_dim + 4) * 4;
    const int misc = (warps * 32 + 1 + warps) * 8 + (4 + warps + 2 * kPackedItems) * 4;  // scan, joins, packed rows
    const int fixed = warps * 2 * partial + warps * 2 * int(sizeof(Record)) + misc;
    int stages = (kSmemBytes - fixed) / (warps * (stage + kTiles * 8));
    stages = stages > 3 ? 3 : stages;
    l.stages = stages;
    l.partials = warps * stages * stage;
    l.records = l.partials + warps * 2 * partial;
    l.meta = l.records + warps * 2 * int(sizeof(Record));
    l.misc = l.meta + warps * stages * kTiles * 8;
    l.total = l.misc + misc;
    return l;
}
static_assert(layout_of(12, 8, 128).stages >= 1 && layout_of(16, 8, 64).stages >= 2 && layout_of(8, 8, 128).stages >= 2);
static_assert(layout_of(12, 8, 128).total <= kSmemBytes && layout_of(16, 1, 64).total <= kSmemBytes);

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// A partial row of one query head: head_dim outputs, then max and sum.
template <int D>
struct Joined {
    float m = -INFINITY, l = 0.f, o[D / 4];
    __device__ __forceinline__ void clear() {
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) o[i] = 0.f;
    }
    // lane (n, c): head n, dims 16 i + 4 c + 0 .. 3
    template <bool kGlobal>
    __device__ __forceinline__ void add(const float* slot, int heads, int lane) {
        const int n = lane >> 2, c = lane & 3;
        if (n >= heads) return;
        const float* row = slot + n * (D + 4);
        float v[D / 4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const float4* at = reinterpret_cast<const float4*>(row + 16 * i + 4 * c);
            const float4 x = kGlobal ? __ldcg(at) : *at;  // other CTAs wrote it: from L2
            v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
        }
        const float2* tail = reinterpret_cast<const float2*>(row + D);
        const float2 ml = kGlobal ? __ldcg(tail) : *tail;
        const float top = fmaxf(m, ml.x);
        const float a = m == top ? 1.f : ex2(m - top), b = ml.x == top ? 1.f : ex2(ml.x - top);
        l = l * a + ml.y * b;
        m = top;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) o[i] = fmaf(o[i], a, v[i] * b);
    }
    __device__ __forceinline__ void store(float* slot, int heads, int lane) const {
        const int n = lane >> 2, c = lane & 3;
        if (n >= heads) return;
        float* row = slot + n * (D + 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            *reinterpret_cast<float4*>(row + 16 * i + 4 * c) =
                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        if (c == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m, l);
    }
    template <class T>
    __device__ __forceinline__ void write(T* out, int heads, int lane) const {
        const int n = lane >> 2, c = lane & 3;
        if (n >= heads) return;
        const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            store4(out + n * D + 16 * i + 4 * c, o[4 * i] * r, o[4 * i + 1] * r, o[4 * i + 2] * r,
                   o[4 * i + 3] * r);
    }
};

template <class T, int F, int D, bool kPacked>
__global__ void __launch_bounds__(warps_of<T, D>() * 32, 1)
    decode_kernel(const AttentionParams p) {
    constexpr int kWarps = warps_of<T, D>(), kThreads = kWarps * 32, kStage = 2 * kUnit * D;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = p.heads / p.cache.kv_heads, subs = (group + 7) / 8, per = p.cache.kv_heads * subs;
    const int slots = min(group, 8);  // partial rows
    const Layout lay = layout_of(kWarps, slots, D);
    const int partial = slots * (D + 4);
    unsigned char* ring = smem + warp * lay.stages * kStage;
    float* partials = reinterpret_cast<float*>(smem + lay.partials);
    Record* records = reinterpret_cast<Record*>(smem + lay.records);
    float2* meta = reinterpret_cast<float2*>(smem + lay.meta) + warp * lay.stages * kTiles;
    int64_t* sums = reinterpret_cast<int64_t*>(smem + lay.misc);  // [kWarps] units of each warp's rows
    int64_t* before = sums + kWarps;                              // [kThreads + 1] units before each thread's rows
    int* joins = reinterpret_cast<int*>(before + kThreads + 1);   // [2] CTAs to join (0: none), [2] their records
    int* longest_of = joins + 4;                                  // [kWarps] most units of a row of each warp
    if (lane < 2) records[2 * warp + lane].units = 0;
    if (tid < 2) joins[tid] = 0;
    pdl_enter();

    // ---- units of all rows (thread t adds up rows t share .. ), and where each warp begins
    const int bt = p.cache.block_tokens;
    const int64_t longest = int64_t(p.table_stride) * bt;
    const int share = (p.count + kThreads - 1) / kThreads;
    // Packed rows: each one's sequence, and tokens up to its position (0: no row, or out of range)
    int *row_tokens = longest_of + kWarps, *row_seq = row_tokens + kPackedItems;
    if constexpr (kPacked) {
        if (tid < p.count) {
            int low = 0, high = p.sequences;  // the first sequence that ends behind the row
            while (low < high) {
                const int i = (low + high) / 2;
                if (p.row_offsets[i + 1] <= tid) {
                    low = i + 1;
                } else {
                    high = i;
                }
            }
            int n = 0;
            if (low < p.sequences) {
                int first, start;
                const int rows = sequence_rows(p, low, first, start);
                if (tid >= first && tid < first + rows) n = start + tid - first + 1;
            }
            row_tokens[tid] = n, row_seq[tid] = low;
        }
        __syncthreads();
    }
    auto table_of = [&](int row) { return p.tables + int64_t(kPacked ? row_seq[row] : row) * p.table_stride; };
    auto tokens = [&](int row) {
        if constexpr (kPacked) return row_tokens[row];
        const int n = p.lengths[row];
        if (n >= 0 && n <= longest) return n;
        raise_error(p.error, kErrBounds);
        return 0;
    };
    auto units_of = [&](int row) { return row < p.count ? int((unsigned(tokens(row)) + kUnit - 1) / kUnit) : 0; };
    // A CTA per item, or equal runs
    int64_t mine = 0;
    int most = 0;
    for (int i = 0; i < share; ++i) {
        const int u = units_of(tid * share + i);
        mine += u, most = max(most, u);
    }
    int64_t upto = mine;  // inclusive scan over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) sums[warp] = upto, longest_of[warp] = most;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, lane < kWarps ? longest_of[lane] : 0);
    bool whole = int64_t(p.count) * per <= int64_t(gridDim.x);
    if (whole) {  // few rows: 32 bits hold their units
        const int all = int(__reduce_add_sync(0xffffffffu, lane < kWarps ? unsigned(sums[lane]) : 0u)) * per;
        whole = most <= all / int(gridDim.x) + kWholeUnits * kWarps;
    }
    int row = 0, item = 0, unit = 0;
    int ctas, cta_units = 0, extra = 0;
    int64_t cta_begin = 0, base = 0;  // CTA c's run: `base` units, one more for the first `extra` CTAs
    if (whole) {
        ctas = p.count * per;
        if (int(blockIdx.x) < ctas) {
            row = blockIdx.x / per, item = blockIdx.x % per;
            cta_units = units_of(row);
        }
    } else {
        int64_t x = lane < warp ? sums[lane] : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        before[tid] = x + upto - mine;
        if (tid == kThreads - 1) before[kThreads] = x + upto;
        __syncthreads();
        const int64_t total = before[kThreads] * per;
        const int64_t want = (total + kWarps * kMinUnits - 1) / (kWarps * kMinUnits);
        ctas = int(want < int64_t(gridDim.x) ? want : int64_t(gridDim.x));
        const int parts = max(ctas, 1);
        base = total >> 32 ? total / parts : int64_t(uint32_t(total) / uint32_t(parts));
        extra = int(total - base * parts);
        if (base >= kMostUnits) {
            raise_error(p.error, kErrBounds);
            return;
        }
        cta_begin = blockIdx.x * base + min(int(blockIdx.x), extra);
        if (int(blockIdx.x) < ctas) cta_units = int(base) + (int(blockIdx.x) < extra);
    }
    auto cta_of = [&](int64_t unit) {
        const int64_t split = extra * (base + 1);
        return int(unit < split ? unit / (base + 1) : extra + (unit - split) / base);
    };
    // the warp's run, likewise
    const int each = cta_units / kWarps, more = cta_units % kWarps, run = each + (warp < more);
    const int64_t begin = cta_begin + warp * each + min(warp, more);
    if (whole) {
        unit = int(begin);
    } else if (run > 0) {
        // the last thread whose rows begin at or before `begin`, then the row among its rows
        int t = (31 - __clz(__ballot_sync(0xffffffffu, before[lane * kWarps] * per <= begin))) * kWarps;
        t += 31 - __clz(__ballot_sync(0xffffffffu, lane < kWarps && before[t + min(lane, kWarps - 1)] * per <= begin));
        row = t * share;
        int64_t at = before[t];
        for (int end = row + share;; row += 32) {  // 32 rows at a time
            const int mine = row + lane < end ? units_of(row + lane) : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, (at + upto) * per > begin);
            if (past) {
                const int i = __ffs(past) - 1;
                const int u = __shfl_sync(0xffffffffu, mine, i);
                const int in = int(begin - (at + __shfl_sync(0xffffffffu, upto, i) - u) * per);
                row += i, item = in / u, unit = in % u;
                break;
            }
            at += __shfl_sync(0xffffffffu, upto, 31);
        }
    }

    // ---- this warp's run. Producer: the next unit to copy, and a window of 32 tiles (block,
    // row, scales) over the lanes
    const int in_page = bt / kTile;
    // 16-byte words of a tile row by row, 32 lanes at a time: kRows rows, kTimes times
    constexpr int kRows = 512 / D, kTimes = kTile / kRows;
    const int to_row = lane / (D / 16);
    uint32_t to[2];  // a row and one kRows further on (which the swizzle may tell apart), words of this lane
#pragma unroll
    for (int i = 0; i < 2; ++i)
        to[i] = smem_u32(ring) + (to_row + i * kRows) * D + swizzled<D>(to_row + i * kRows, lane % (D / 16)) * 16;
    int c_row = row, c_item = item, c_unit = unit, c_left = run, c_len = run ? tokens(row) : 0;
    int w_next = 16;                       // unit of the window that comes next
    const unsigned char* w_at = nullptr;   // this lane's tile (K; V is one block of rows on)
    float2 w_scale{};
    {
        auto issue = [&](int stage) {
            if (c_left) {
                if (w_next == 16) {
                    w_next = 0;
                    const int tile = kTiles * c_unit + lane;
                    w_scale = make_float2(0.f, 0.f);
                    if (tile * kTile < c_len && lane < kTiles * c_left) {
                        const int kh = c_item / subs;
                        const int block = block_id(p.cache, table_of(c_row), p.table_stride, tile / in_page, p.error);
                        w_scale = *reinterpret_cast<const float2*>(p.cache.scales + block * p.cache.scale_stride + 2 * kh);
                        w_at = p.cache.pages + tile_offset(p.cache, block, kh, 0, D) + tile % in_page * (kTile * D);
                    }
                }
                if (lane >> 1 == w_next) meta[kTiles * stage + (lane & 1)] = w_scale;
#pragma unroll
                for (int u = 0; u < kTiles; ++u) {
                    const unsigned char* from = reinterpret_cast<const unsigned char*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(w_at), kTiles * w_next + u)) + lane * 16;
                    if ((kTiles * c_unit + u) * kTile >= c_len) break;
#pragma unroll
                    for (int i = 0; i < kTimes; ++i) {
                        const uint32_t at = to[i & 1] + stage * kStage + u * (kStage / 2) + (i >> 1) * (2 * kRows * D);
                        copy16(at, from + i * 512);
                        copy16(at + kTile * D, from + bt * D + i * 512);
                    }
                }
                ++w_next, ++c_unit, --c_left;
                if (c_unit * kUnit >= c_len && c_left) {
                    c_unit = 0, w_next = 16;
                    if (++c_item == per) {
                        c_item = 0;
                        do c_len = tokens(++c_row);
                        while (c_len == 0);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");  // one per unit, empty ones included
        };
        for (int s = 0; s < lay.stages; ++s) issue(s);
        __syncwarp();

        // rows without tokens, while the copies fly
        // (packed: sequences that no row was found in have their metadata checked too)
        for (int r = blockIdx.x * kThreads + tid, at, from; kPacked && r < p.sequences; r += gridDim.x * kThreads)
            sequence_rows(p, r, at, from);
        for (int r = blockIdx.x * kWarps + warp; !kPacked && r < p.count; r += gridDim.x * kWarps)
            if (tokens(r) == 0) {
                T* out = static_cast<T*>(p.out) + r * p.out_stride;
                for (int i = lane; i < p.heads * D / 4; i += 32) store4(out + 4 * i, 0.f, 0.f, 0.f, 0.f);
            }
        if (int(blockIdx.x) >= ctas) return;

        const int k_row = WarpRow<T, F, D>::token(0, lane >> 2);                    // and 8 rows on
        const int v_row = WarpRow<T, F, D>::token((lane >> 3) & 1, lane & 7);       // this lane's matrix row
        int stage = 0, emitted = 0;
        for (int done = 0; done < run;) {
            const int len = tokens(row), units = (len + kUnit - 1) / kUnit;
            const int last = min(units, unit + run - done), from = unit;
            const int kh = item / subs, sub = item % subs;
            const int h0 = kh * group + sub * 8, heads = min(8, group - sub * 8);
            WarpRow<T, F, D> w;
            w.begin(static_cast<const T*>(p.q) + row * p.q_stride + h0 * D, heads, p.scale, lane);
            for (; unit < last; ++unit) {
                if (lay.stages == 3) {
                    asm volatile("cp.async.wait_group 2;" ::: "memory");
                } else if (lay.stages == 2) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                } else {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                }
                __syncwarp();
                const unsigned char* at = ring + stage * kStage;
                auto load_k = [&](int u, int i, int h) {
                    return *reinterpret_cast<const uint4*>(at + (2 * u * kTile + k_row + 8 * i) * D +
                                                           swizzled<D>(k_row, 4 * h + (lane & 3)) * 16);
                };
                const uint32_t v_at = smem_u32(at) + (kTile + v_row) * D;
                auto load_v = [&](int u, int q, uint32_t (&r)[4]) {
                    load_transposed(r, v_at + 2 * u * kTile * D + swizzled<D>(v_row, 2 * q + (lane >> 4)) * 16);
                };
                float2 scale[kTiles];
#pragma unroll
                for (int u = 0; u < kTiles; ++u) scale[u] = meta[kTiles * stage + u];
                if (len - unit * kUnit >= kUnit) {
                    w.template step<false>(load_k, load_v, scale, kUnit, lane);
                } else {
                    w.template step<true>(load_k, load_v, scale, len - unit * kUnit, lane);
                }
                if (!WarpRow<T, F, D>::kSplit && (unit + 1) % WarpRow<T, F, D>::kChain == 0) w.close();
                __syncwarp();
                issue(stage);
                if (++stage == lay.stages) stage = 0;
            }
            w.end();
            done += last - from;
            if (from == 0 && last == units) {
                w.write(static_cast<T*>(p.out) + row * p.out_stride + h0 * D, heads, lane);
            } else {
                Joined<D> j;
                j.m = w.m, j.l = w.l;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) j.o[4 * (i / 2) + i % 2] = w.o[i][0], j.o[4 * (i / 2) + i % 2 + 2] = w.o[i][1];
                j.store(partials + (2 * warp + emitted) * partial, slots, lane);
                if (lane == 0)
                    records[2 * warp + emitted] = {begin + done - last, row, item, units, from == 0, last == units};
                ++emitted;
            }
            unit = 0;
            if (done < run && ++item == per) {
                item = 0;
                do ++row;
                while (tokens(row) == 0);
            }
        }
    }
    __syncthreads();

    // ---- join the warps' partials: the warp of an item's first record in this CTA joins them
    float* store = reinterpret_cast<float*>(static_cast<unsigned char*>(p.workspace) + kCounterBytes);
    unsigned* counters = static_cast<unsigned*>(p.workspace);
    auto same = [&](const Record& a, const Record& b) { return b.units && a.row == b.row && a.item == b.item; };
    auto output = [&](const Record& r) {
        return static_cast<T*>(p.out) + r.row * p.out_stride + (r.item / subs * group + r.item % subs * 8) * D;
    };
    auto heads_of = [&](const Record& r) { return min(8, group - r.item % subs * 8); };
    for (int k = 0; k < 2; ++k) {
        const int index = 2 * warp + k;
        const Record r = records[index];
        if (!r.units) continue;
        int previous = index - 1;
        while (previous >= 0 && !records[previous].units) --previous;
        if (previous >= 0 && same(r, records[previous])) continue;
        Joined<D> j;
        j.clear();
        int ends = 0;
        for (int i = index; i < 2 * kWarps; ++i) {
            if (!records[i].units) continue;
            if (!same(r, records[i])) break;
            j.template add<false>(partials + i * partial, slots, lane);
            ends = records[i].ends;
        }
        if (r.begins && ends) {
            j.write(output(r), heads_of(r), lane);
            continue;
        }
        // 0: the item began in an earlier CTA, 1: it begins here
        j.store(store + (int64_t(blockIdx.x) * 2 + r.begins) * partial, slots, lane);
        __threadfence();
        __syncwarp();
        if (lane == 0) {
            const int c0 = cta_of(r.first), n = cta_of(r.first + r.units - 1) - c0 + 1;
            if (atomicAdd(counters + c0, 1u) == unsigned(n - 1)) {
                counters[c0] = 0;
                joins[r.begins] = n;
                records[index].begins = c0 + 1;  // read back below as the joining record
                joins[2 + r.begins] = index;
            }
            __threadfence();
        }
    }
    __syncthreads();

    // ---- join the CTAs' partials, all warps at once
    float* level = reinterpret_cast<float*>(smem);  // the rings are empty
    for (int k = 0; k < 2; ++k) {
        const int n = joins[k];
        if (n == 0) continue;
        const Record r = records[joins[2 + k]];
        const int c0 = r.begins - 1;
        Joined<D> j;
        j.clear();
        for (int i = warp; i < n; i += kWarps) j.template add<true>(store + (int64_t(c0 + i) * 2 + (i == 0)) * partial, slots, lane);
        j.store(level + warp * partial, slots, lane);
        __syncthreads();
        if (warp == 0) {
            j.clear();
            for (int i = 0; i < min(n, kWarps); ++i) j.template add<false>(level + i * partial, slots, lane);
            j.write(output(r), heads_of(r), lane);
        }
        __syncthreads();
    }
}

}  // namespace

size_t decode_workspace(int group, int head_dim) {
    return kCounterBytes + size_t(kCtas) * 2 * (group < 8 ? group : 8) * (head_dim + 4) * 4;
}

template <bool kPacked>
static cudaError_t launch(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    return dispatch(type, format, head_dim, [&](auto t, auto f, auto d) {
        using T = decltype(t);
        constexpr int kDim = decltype(d)::value, kWarps = warps_of<T, kDim>();
        auto kernel = decode_kernel<T, decltype(f)::value, kDim, kPacked>;
        const int group = p.heads / p.cache.kv_heads;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return e;
        return launch_pdl(kernel, dim3(kCtas), dim3(kWarps * 32), size_t(layout_of(kWarps, group < 8 ? group : 8, kDim).total),
                          stream, p);
    });
}

cudaError_t launch_decode(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    return launch<false>(p, type, format, head_dim, stream);
}

cudaError_t launch_packed(AttentionParams p, int type, int format, int head_dim, cudaStream_t stream) {
    p.sequences = p.count, p.count = p.rows;
    return launch<true>(p, type, format, head_dim, stream);
}

}  // namespace kv8
}  // namespace mpb
