// Attention of one query row (up to 8 query heads of one kv head) by one warp over
// units of 16 tokens of the 8-bit cache, on warp-level tensor ops (sm_100a).
//
// Scores: S = Q K^T as m16n8k16 products. Rows 0..7 of A are the FP16 high halves of
// the 8 heads' queries, rows 8..15 their low halves; B's columns are 8 tokens. The codes
// are exact in FP16, so hi + lo rows give FP32-level scores from one product. Lane (n,
// c) = (lane / 4, lane % 4) holds B's column n: the 16 bytes c of token n's row (the K
// dimension is permuted the same way in A, so each lane's load is one 16-byte word).
// Weights: lane (n, c) then owns head n's scores of tokens 2c, 2c + 1 of each 8, which is
// the A layout of the second product, P V; V, read like K, is transposed by movmatrix.
// V's block scale is folded into the weights.
//
// Tensor-op sums are cut, not rounded: each added unit loses about 2^-25.7 of the sum
// (measured: 1.8e-5 after 1000 units). FP32 outputs therefore add the products up in
// chains of kChain units and the chains in FP32 registers.
//
// The state is a running softmax: m (largest score), l (sum of weights), and outputs in
// units of `unit`, the largest weight times scale so far (moved whenever m moves or a
// larger product comes), so that the weights fill FP16's range.
#pragma once
#include "kv8.cuh"

namespace mpb {
namespace kv8 {

constexpr int kUnit = 16;                  // tokens of a unit
constexpr int kChain = 8;                  // units per chain of tensor-op sums (FP32 outputs)
constexpr float kWeightTop = 4096.f;       // weights are at most 2^12 in FP16
constexpr float kUnitFloor = 7.7e-34f;     // 2^-110: below every scale the append makes

template <class T, int F, int D>
struct WarpRow {
    static constexpr int kHalves = D / 64;
    static constexpr bool kSplit = sizeof(T) == 4;  // BF16 outputs: weights as one FP16 half (2^-12 relative)
    uint32_t qa[D / 16][4];
    float o[D / 8][4];  // [tile][0, 1: hi rows; 2, 3: lo rows]
    float sum[kSplit ? D / 8 : 1][2];  // finished chains
    float m, l, unit, inv_unit, k_factor;
    int chain;

    // Query heads h0 .. h0 + heads - 1 at `q` (head stride D); absent heads are zero.
    __device__ __forceinline__ void begin(const T* q, int heads, float scale, int lane) {
        const int n = lane >> 2, c = lane & 3;
        float v[D / 4];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (n < heads) load4(q + n * D + (i >> 2) * 64 + c * 16 + (i & 3) * 4, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j], amax = fmaxf(amax, fabsf(x[j]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float factor, inverse;
        row_factor(amax, factor, inverse);
        k_factor = inverse * scale * kLog2e;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            split_pair(v[4 * i] * factor, v[4 * i + 1] * factor, qa[i][0], qa[i][1]);
            split_pair(v[4 * i + 2] * factor, v[4 * i + 3] * factor, qa[i][2], qa[i][3]);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < (kSplit ? D / 8 : 1); ++i) sum[i][0] = sum[i][1] = 0.f;
        m = -INFINITY, l = 0.f, unit = kUnitFloor, inv_unit = kWeightTop / kUnitFloor, chain = 0;
    }

    // One unit. k, v: [half][token n, token 8 + n] 16-byte words of this lane; tokens at
    // or past `valid` (1 .. 16) are masked.
    __device__ __forceinline__ void step(uint4 (&k)[kHalves][2], uint4 (&v)[kHalves][2], float ks, float vs, int valid,
                                         int lane) {
        const int n = lane >> 2, c = lane & 3;
        if (valid < kUnit) {  // bytes behind the last token may be NaN codes
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (8 * i + n >= valid) {
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) k[h][i] = v[h][i] = make_uint4(0, 0, 0, 0);
                }
        }
        float s[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const uint32_t w[4] = {k[h][i].x, k[h][i].y, k[h][i].z, k[h][i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t b0, b1;
                    widen4<F>(w[j], b0, b1);
                    mma16816(acc, qa[4 * h + j], b0, b1);
                }
            }
            s[i][0] = acc[0] + acc[2];
            s[i][1] = acc[1] + acc[3];
        }
        const float f = k_factor * ks;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) top = fmaxf(top, 8 * i + 2 * c + j < valid ? s[i][j] * f : -INFINITY);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(m, top);
        const float reach = m_new == -INFINITY ? 0.f : vs * ex2(top - m_new);  // largest weight times scale here
        if (__any_sync(0xffffffffu, top > m || reach > unit)) {
            const float decay = m_new == -INFINITY ? 1.f : ex2(m - m_new);
            const float unit_new = fmaxf(fmaxf(unit * decay, reach), kUnitFloor);
            const float move = decay * unit / unit_new;
            l *= decay;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] *= move;
                if constexpr (kSplit) sum[i][0] *= move, sum[i][1] *= move;
            }
            m = m_new, unit = unit_new, inv_unit = kWeightTop / unit_new;
        }
        const float base = m == -INFINITY ? 0.f : m, w = vs * inv_unit;
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float p0 = 8 * i + 2 * c < valid ? ex2(fmaf(s[i][0], f, -base)) : 0.f;
            const float p1 = 8 * i + 2 * c + 1 < valid ? ex2(fmaf(s[i][1], f, -base)) : 0.f;
            l += p0 + p1;
            if constexpr (kSplit) {
                split_pair(p0 * w, p1 * w, a[2 * i], a[2 * i + 1]);
            } else {
                const __half2 h = __floats2half2_rn(p0 * w, p1 * w);
                a[2 * i] = *reinterpret_cast<const uint32_t*>(&h);
                a[2 * i + 1] = 0;
            }
        }
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const uint32_t w0[4] = {v[h][0].x, v[h][0].y, v[h][0].z, v[h][0].w};
            const uint32_t w1[4] = {v[h][1].x, v[h][1].y, v[h][1].z, v[h][1].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t x0, x1, y0, y1;
                widen4<F>(w0[j], x0, x1);
                widen4<F>(w1[j], y0, y1);
                mma16816(o[8 * h + 2 * j], a, transpose8x8(x0), transpose8x8(y0));
                mma16816(o[8 * h + 2 * j + 1], a, transpose8x8(x1), transpose8x8(y1));
            }
        }
        if constexpr (kSplit) {
            if (++chain == kChain) {
                close();
                chain = 0;
            }
        }
    }

    __device__ __forceinline__ void close() {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            sum[i][0] += o[i][0] + o[i][2];
            sum[i][1] += o[i][1] + o[i][3];
            o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
    }

    // Sum of weights over the head's lanes; o[..][0, 1] become the head's outputs in plain
    // units (unnormalised). Afterwards lane (n, c) holds head n's dims
    // (i / 8) * 64 + 16 c + 2 (i % 8) + {0, 1} in o[i][0, 1].
    __device__ __forceinline__ void end() {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float u = unit * (1.f / kWeightTop);
        if constexpr (kSplit) close();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            o[i][0] = (kSplit ? sum[i][0] : o[i][0] + o[i][2]) * u;
            o[i][1] = (kSplit ? sum[i][1] : o[i][1] + o[i][3]) * u;
        }
    }

    // out (head stride D) = o / l; a row without tokens (l = 0) is zero.
    __device__ __forceinline__ void write(T* out, int heads, int lane) const {
        const int n = lane >> 2, c = lane & 3;
        if (n >= heads) return;
        const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < D / 8; i += 2)
            store4(out + n * D + (i >> 3) * 64 + c * 16 + (i & 7) * 2, o[i][0] * r, o[i][1] * r, o[i + 1][0] * r,
                   o[i + 1][1] * r);
    }
};

}  // namespace kv8
}  // namespace mpb
