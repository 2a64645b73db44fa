// mp_kv8_attention_prefill: causal attention of packed chunks of rows over the 8-bit paged cache.
#include "kv8_warp.cuh"

namespace mpb {
namespace kv8 {
namespace {

constexpr int kThreads = 128;

// One warp per (row, kv head, 8 query heads), token unit by token unit.
template <class T, int F, int D>
__global__ void __launch_bounds__(kThreads) row_kernel(const AttentionParams p) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int group = p.heads / p.cache.kv_heads, subs = (group + 7) / 8;
    const int64_t item = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    const int per = p.cache.kv_heads * subs;
    const int row = int(item / per), kh = int(item % per) / subs, sub = int(item % per) % subs;
    if (row >= p.rows) return;
    const int bt = p.cache.block_tokens;
    int before = 0;
    for (int i = lane; i < p.count; i += 32) before += p.row_offsets[i + 1] <= row;
    const int seq = __reduce_add_sync(0xffffffffu, before);
    if (seq >= p.count) return;
    const int begin = p.row_offsets[seq], start = p.starts[seq];
    const int64_t end = int64_t(start) + row - begin + 1;
    if (row < begin || start < 0 || end > int64_t(p.table_stride) * bt) {
        if (lane == 0) raise_error(p.error, kErrBounds);
        return;
    }
    const int len = int(end);
    const int h0 = kh * group + sub * 8, heads = min(8, group - sub * 8);
    WarpRow<T, F, D> w;
    w.begin(static_cast<const T*>(p.q) + row * p.q_stride + h0 * D, heads, p.scale, lane);
    const int32_t* table = p.tables + int64_t(seq) * p.table_stride;
    const int n = lane >> 2, c = lane & 3;
    for (int t = 0; t < len; t += kUnit) {
        const unsigned char* at[kTiles];
        float2 scale[kTiles];
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            const int token = t + u * kTile;
            scale[u] = make_float2(0.f, 0.f);
            at[u] = at[0];
            if (token < len) {
                const int block = block_id(p.cache, table, p.table_stride, token / bt, p.error);
                scale[u] = *reinterpret_cast<const float2*>(p.cache.scales + block * p.cache.scale_stride + 2 * kh);
                at[u] = p.cache.pages + tile_offset(p.cache, block, kh, 0, D) + (token % bt) * D;
            }
        }
        auto load_k = [&](int u, int i, int h) {
            return *reinterpret_cast<const uint4*>(at[u] + w.token(i, n) * D + h * 64 + c * 16);
        };
        auto load_v = [&](int u, int q, uint32_t (&r)[4]) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                r[g] = transpose8x8(*reinterpret_cast<const uint32_t*>(at[u] + (bt + w.token(g & 1, n)) * D + 32 * q +
                                                                       16 * (g >> 1) + 4 * c));
        };
        if (len - t >= kUnit) {
            w.template step<false>(load_k, load_v, scale, kUnit, lane);
        } else {
            w.template step<true>(load_k, load_v, scale, len - t, lane);
        }
    }
    w.end();
    w.write(static_cast<T*>(p.out) + row * p.out_stride + h0 * D, heads, lane);
}

}  // namespace

size_t prefill_workspace(int, int) { return 256; }

cudaError_t launch_prefill(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    const int64_t items = int64_t(p.rows) * p.cache.kv_heads * ((p.heads / p.cache.kv_heads + 7) / 8);
    return dispatch(type, format, head_dim, [&](auto t, auto f, auto d) {
        return launch_pdl(row_kernel<decltype(t), decltype(f)::value, decltype(d)::value>,
                          dim3(unsigned((items + 3) / 4)), dim3(kThreads), 0, stream, p);
    });
}

}  // namespace kv8
}  // namespace mpb
