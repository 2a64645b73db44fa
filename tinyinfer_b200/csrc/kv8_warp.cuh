// Attention of one query row (up to 8 query heads of one kv head) by one warp over
// units of 32 tokens (two tiles of 16, each in one block) of the 8-bit cache, on
// warp-level tensor ops (sm_100a).
//
// Scores: S = Q K^T as m16n8k16 products. Rows 0..7 of A are the FP16 high halves of
// the 8 heads' queries, rows 8..15 their low halves; B's columns are 8 tokens. The codes
// are exact in FP16, so hi + lo rows give FP32-level scores from one product. Lane (n,
// c) = (lane / 4, lane % 4) holds B's column n: the 16 bytes c of token n's row (the K
// dimension is permuted the same way in A, so each lane's load is one 16-byte word).
// Weights: lane (n, c) then owns head n's scores of tokens 2c, 2c + 1 of each 8, which is
// the A layout of the second product, P V. Its B wants two tokens of one dim side by side:
// V's bytes are read as 16-bit elements (two dims) in transposed 8 x 8 matrices, which gives
// a lane two dims of two tokens. (A first version transposed the widened halves with
// movmatrix: the pipe that it shares with exp2 took 660 cycles a unit, four times the rest.)
// V's block scale is folded into the weights.
//
// Tensor-op sums are cut, not rounded: each added tile loses about 2^-25.7 of the sum
// (measured: 1.8e-5 after 1000 tiles; up to 2^-23). Outputs are therefore added up in chains of
// kChain units, and the chains in FP32 registers: 128 tokens a chain for FP32 outputs, 32768
// (2048 tiles, at most 2.4e-4) for BF16 ones, which came out 6e-3 small after one chain of 2^20.
// The sum of weights goes by the same chains (in one, 2^20 weights of 0.7 were 1e-3 off).
//
// The state is a running softmax: m (the reference score), l (sum of weights), and outputs
// in units of `unit`, a power of two at most the largest weight times scale so far (but see
// kUnitFloor and kScaleFloor), so that the weights fill FP16's range. FP16 has room for weights
// 2^7 times 2^8 (`unit` is below the largest by up to 2), so m and unit move only when a score
// passes m by 6 (in powers of two) or a scale reaches twice the unit: moving them every time that
// the maximum grew cost a fifth of the instructions. FP16's smallest half step, 2^-25, is 2^-33
// of the largest.
#pragma once
#include "kv8.cuh"

namespace mpb {
namespace kv8 {

constexpr int kTile = 16;                  // tokens of a tile: the K of one product
constexpr int kTiles = 2;                  // tiles of a unit: their products overlap, and votes and shuffles halve
constexpr int kUnit = kTile * kTiles;
constexpr float kWeightTop = 256.f;        // a weight of `unit` is 2^8 in FP16
constexpr float kSlack = 6.f;              // a score may pass m by this (weights up to 2^6)
constexpr float kUnitFloor = 7.70371977754894e-34f;  // 2^-110: below every scale the append makes
// 2^-118: `unit` is at least that much of a scale in use (so far as reach < 2 unit: 2^-119), so that
// kWeightTop * scale / unit stays below 2^127 when the tokens under a large scale have faint weights
constexpr float kScaleFloor = 3.0092655e-36f;

template <class T, int F, int D>
struct WarpRow {
    static constexpr int kHalves = D / 64;
    static constexpr bool kSplit = sizeof(T) == 4;  // BF16 outputs: weights as one FP16 half (2^-12 relative)
    static constexpr int kChain = kSplit ? 4 : 1024;  // units per chain of tensor-op sums (the caller ends BF16's)
    uint32_t qa[D / 16][4];
    // outputs: lane (n, c) holds head n's dims 16 i / 2 + 4 c + i % 2 + {0, 2} in o[i][0, 1]
    // (weights' hi halves) and o[i][2, 3] (lo; BF16: finished chains, to which the products add zeros)
    float o[D / 8][4];
    float sum[kSplit ? D / 8 : 1][2];  // finished chains
    float m, l, chain_l, unit, inv_unit, k_factor;  // chain_l: of the sum of weights, the chain's part
    int chain;

    // Token of column x of 8 in half `i` of a tile. 128-byte rows: columns 2i and 2i + 1 are
    // four rows apart, so that the swizzled chunks which 8 lanes read lie in different banks.
    static __device__ __forceinline__ int token(int i, int x) { return 8 * i + (D == 128 ? (x >> 1) + 4 * (x & 1) : x); }

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
        m = -INFINITY, l = chain_l = 0.f, unit = kUnitFloor, inv_unit = kWeightTop / kUnitFloor, chain = 0;
    }

    // One unit. load_k(u, i, h): the 16-byte word c of 64-byte half h of token(i, n)'s row in
    // tile u (bytes behind the last token may be NaN codes: they become zero); load_v(u, q, r):
    // dims 32 q .. 32 q + 31 of V's tile u as four transposed matrices, r[2 a + i] = chunk 2 q + a
    // of the tokens of half i; scale[u]: the K and V scales. kLast: tokens at or past `valid`
    // (1 .. 32) are masked (a tile without tokens has scales 0); else all 32 are there.
    template <bool kLast, class LoadK, class LoadV>
    __device__ __forceinline__ void step(LoadK load_k, LoadV load_v, const float2 (&scale)[kTiles], int valid, int lane) {
        const int n = lane >> 2, c = lane & 3;
        float acc[kTiles][2][4];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            uint4 k[kTiles][2];
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    k[u][i] = load_k(u, i, h);
                    if (kLast && u * kTile + token(i, n) >= valid) k[u][i] = make_uint4(0, 0, 0, 0);
                    if (h == 0) acc[u][i][0] = acc[u][i][1] = acc[u][i][2] = acc[u][i][3] = 0.f;
                }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < kTiles; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 w = k[u][i];
                        uint32_t b0, b1;
                        widen4<F>(j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w, b0, b1);
                        mma16816(acc[u][i], qa[4 * h + j], b0, b1);
                    }
        }
        float t[kTiles][2][2];
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            const float f = k_factor * scale[u].x;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                t[u][i][0] = (acc[u][i][0] + acc[u][i][2]) * f;
                t[u][i][1] = (acc[u][i][1] + acc[u][i][3]) * f;
            }
        }
        auto live = [&](int u, int i, int j) { return u * kTile + token(i, 2 * c + j) < valid; };
        if constexpr (kLast) {
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) t[u][i][j] = live(u, i, j) ? t[u][i][j] : -INFINITY;
        }
        float top = -INFINITY, most = 0.f;
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            top = fmaxf(top, fmaxf(fmaxf(t[u][0][0], t[u][0][1]), fmaxf(t[u][1][0], t[u][1][1])));
            most = fmaxf(most, scale[u].y);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m + kSlack || most >= 2.f * unit)) move(t, scale, top);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            const float w = scale[u].y * inv_unit;
            uint32_t a[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float p0 = ex2(t[u][i][0] - base), p1 = ex2(t[u][i][1] - base);
                chain_l += p0 + p1;
                if constexpr (kSplit) {
                    split_pair(p0 * w, p1 * w, a[2 * i], a[2 * i + 1]);
                } else {
                    const __half2 h = __floats2half2_rn(p0 * w, p1 * w);
                    a[2 * i] = *reinterpret_cast<const uint32_t*>(&h);
                    a[2 * i + 1] = 0;
                }
            }
            uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
            if constexpr (kLast)
#pragma unroll
                for (int i = 0; i < 2; ++i) keep[i] = (live(u, i, 0) ? 0xffffu : 0u) | (live(u, i, 1) ? 0xffff0000u : 0u);
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
                uint32_t r[4];
                load_v(u, q, r);
                if constexpr (kLast) r[0] &= keep[0], r[1] &= keep[1], r[2] &= keep[0], r[3] &= keep[1];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t x0, x1, y0, y1;
                    widen_pairs<F>(r[2 * g], x0, x1);
                    widen_pairs<F>(r[2 * g + 1], y0, y1);
                    mma16816(o[4 * q + 2 * g], a, x0, y0);
                    mma16816(o[4 * q + 2 * g + 1], a, x1, y1);
                }
            }
        }
        if constexpr (kSplit) {
            if (++chain == kChain) {
                close();
                chain = 0;
            }
        }
    }

    // Takes the largest score as the reference and the largest weight times scale as the unit,
    // if a head needs it.
    __device__ __forceinline__ void move(const float (&t)[kTiles][2][2], const float2 (&scale)[kTiles], float top) {
        const float m_new = fmaxf(m, top);
        float reach = 0.f;  // largest weight times scale of the unit
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            reach = fmaxf(reach, scale[u].y * kScaleFloor);
            const float tops = fmaxf(fmaxf(t[u][0][0], t[u][0][1]), fmaxf(t[u][1][0], t[u][1][1]));
            if (tops != -INFINITY) reach = fmaxf(reach, scale[u].y * ex2(tops - m_new));
        }
        reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 1));
        reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 2));
        if (!__any_sync(0xffffffffu, top > m + kSlack || reach >= 2.f * unit)) return;
        const float decay = m_new == -INFINITY ? 1.f : ex2(m - m_new);
        const float largest = fminf(fmaxf(fmaxf(unit * decay, reach), kUnitFloor), 8.507059e37f);
        const int exponent = (__float_as_int(largest) >> 23) - 127;  // rounded down to a power of two
        const float by = decay * (unit * pow2(-exponent));
        l *= decay, chain_l *= decay;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] *= by;
            if constexpr (kSplit) sum[i][0] *= by, sum[i][1] *= by;
        }
        m = m_new, unit = pow2(exponent), inv_unit = kWeightTop * pow2(-exponent);
    }

    // Ends a chain.
    __device__ __forceinline__ void close() {
        l += chain_l, chain_l = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            if constexpr (kSplit) {
                sum[i][0] += o[i][0] + o[i][2];
                sum[i][1] += o[i][1] + o[i][3];
                o[i][2] = o[i][3] = 0.f;
            } else {
                o[i][2] += o[i][0];
                o[i][3] += o[i][1];
            }
            o[i][0] = o[i][1] = 0.f;
        }
    }

    // Sum of weights over the head's lanes; o[i][0, 1] become the head's outputs in plain
    // units (unnormalised).
    __device__ __forceinline__ void end() {
        close();
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float u = unit * (1.f / kWeightTop);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            o[i][0] = (kSplit ? sum[i][0] : o[i][2]) * u;
            o[i][1] = (kSplit ? sum[i][1] : o[i][3]) * u;
        }
    }

    // out (head stride D) = o / l; a row without tokens (l = 0) is zero.
    __device__ __forceinline__ void write(T* out, int heads, int lane) const {
        const int n = lane >> 2, c = lane & 3;
        if (n >= heads) return;
        const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < D / 8; i += 2)
            store4(out + n * D + 8 * i + 4 * c, o[i][0] * r, o[i + 1][0] * r, o[i][1] * r, o[i + 1][1] * r);
    }
};

}  // namespace kv8
}  // namespace mpb
