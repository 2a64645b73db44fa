// mp_kv8_append: rotate q and k, quantise k and v, write the 8-bit pages (sm_100a).
//
// Rotation of a pair (a, b) at position p with c = cos[p][i], s = sin[p][i]: (a c - b s,
// b c + a s), the reference's rope_append step (miniprefix/src/backend/cuda/
// llama_runner.cu:20-32). A code is the nearest multiple of the block's scale, so a
// rotated value next to the border of two codes must not be rounded on the way: the
// products of two floats are exact in 64 bits, and the sum is rounded there once.
//
// The unit of work is (block, kv head, K or V): its scale needs the largest magnitude of
// all its new tokens, so one warp takes a whole tile, twice (magnitude, then codes; the
// second read hits L1).
#include "kv8.cuh"

namespace mpb {
namespace kv8 {
namespace {

constexpr int kThreads = 128;

// double -> float rounded to odd, so that a later rounding to fewer bits equals one
// rounding of the double.
__device__ __forceinline__ float to_odd(double x) {
    const float f = __double2float_rz(x);
    return double(f) == x || isnan(x) ? f : __int_as_float(__float_as_int(f) | 1);
}

__device__ __forceinline__ float rounded(double x, float) { return __double2float_rn(x); }
__device__ __forceinline__ float rounded(double x, __nv_bfloat16) { return to_odd(x); }  // store4 rounds it

// A lane's eight values of one head row: two groups of four, at i0 and i1. Chunk c of
// the rotated dims holds four whole pairs; later chunks pass through.
struct Chunk {
    int i0, i1, pair;  // pair: index of the first of the four rotation pairs, -1: none
};
__device__ __forceinline__ Chunk chunk_of(int c, int rotary, int interleaved) {
    if (8 * c >= rotary) return {8 * c, 8 * c + 4, -1};
    return interleaved ? Chunk{8 * c, 8 * c + 4, 4 * c} : Chunk{4 * c, rotary / 2 + 4 * c, 4 * c};
}

// The chunk's eight values, rotated by row `position` of the tables, in 64 bits.
template <class T>
__device__ __forceinline__ void load_rotated(const T* row, Chunk ch, int interleaved, const float* cos,
                                             const float* sin, int rotary, int position, double (&r)[8]) {
    float x[4], y[4];
    load4(row + ch.i0, x);
    load4(row + ch.i1, y);
    if (ch.pair < 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = x[i], r[4 + i] = y[i];
        return;
    }
    float c[4], s[4];
    const size_t at = size_t(position) * (rotary / 2) + ch.pair;
    load4(cos + at, c);
    load4(sin + at, s);
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = i < 2 ? x[2 * i] : y[2 * i - 4], b = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
            r[2 * i] = a * double(c[i]) - b * double(s[i]);
            r[2 * i + 1] = b * double(c[i]) + a * double(s[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = x[i], b = y[i];
            r[i] = a * double(c[i]) - b * double(s[i]);
            r[4 + i] = b * double(c[i]) + a * double(s[i]);
        }
    }
}

// Exponent of the smallest power of two that holds `amax` (finite): 127 = 0.9921875 *
// 2^7 for INT8, 448 = 1.75 * 2^8 for E4M3; at least 2^-100.
template <int F>
__device__ __forceinline__ int scale_exponent(float amax) {
    const int e = (__float_as_int(amax) >> 23) - 127, m = __float_as_int(amax) & 0x7fffff;
    // amax = (1 + m / 2^23) * 2^e; the limit is 1.984375 * 2^6 or 1.75 * 2^8
    const int x = F == MP_KV8_INT8 ? e - 6 + (m > 0x7e0000) : e - 8 + (m > 0x600000);
    return max(x, -100);
}

// Four values in units of the scale as codes.
template <int F>
__device__ __forceinline__ uint32_t encode4(const double (&r)[8], int at, double inv) {
    uint32_t w = 0;
    if constexpr (F == MP_KV8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double y = r[at + i] * inv;
            const int c = isnan(y) ? 0 : __double2int_rn(fmin(fmax(y, -127.0), 127.0));
            w |= uint32_t(c & 255) << (8 * i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float a = to_odd(r[at + i] * inv), b = to_odd(r[at + i + 1] * inv);
            a = isnan(a) ? 0.f : a, b = isnan(b) ? 0.f : b;
            uint16_t h;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(b), "f"(a));
            w |= uint32_t(h) << (8 * i);
        }
    }
    return w;
}

// Four held codes times `ratio` (a power of two below 1), rounded to codes again.
template <int F>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
    uint32_t lo, hi;
    widen4<F>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    const double r[8] = {a.x, a.y, b.x, b.y, 0, 0, 0, 0};
    return encode4<F>(r, 0, double(ratio));
}

template <class T, int F, int D>
__device__ __forceinline__ void append_tile(const AppendParams& p, const T* rows, int64_t stride, int head, int part,
                                            int block, int slot0, int n, int position, int lane) {
    constexpr int kLanes = D / 8;        // lanes of one token
    constexpr int kStep = 32 / kLanes;   // tokens a warp reads at once
    const int c = lane % kLanes, sub = lane / kLanes;
    const int rotary = part ? 0 : p.rotary_dim;
    const Chunk ch = chunk_of(c, rotary, p.interleaved);
    const T* at = rows + head * D;
    float amax = 0.f;
    bool odd = false;
    for (int t = sub; t < n; t += kStep) {
        double r[8];
        load_rotated(at + t * stride, ch, p.interleaved, p.cos, p.sin, rotary, position + t, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = fabsf(__double2float_rn(r[i]));
            const bool finite = f <= 3.402823466e38f;
            odd |= !finite;
            amax = finite ? fmaxf(amax, f) : amax;
        }
    }
    amax = warp_max(amax);
    int x = scale_exponent<F>(amax);
    float* scale = p.cache.scales + int64_t(block) * p.cache.scale_stride + head * 2 + part;
    unsigned char* tile = p.cache.pages + tile_offset(p.cache, block, head, part, D);
    if (slot0 > 0) {
        const float held = *scale;
        const int bits = __float_as_int(held), e = (bits >> 23) - 127;
        if ((bits & 0x807fffff) != 0 || e < -126 || e > 127) {
            odd = true;  // not a power of two: the held codes stay as they are under the new scale
        } else if (e >= x) {
            x = e;
        } else {
            const float ratio = e - x < -126 ? 0.f : pow2(e - x);
            for (int i = lane; i < slot0 * D / 16; i += 32) {
                uint4* w = reinterpret_cast<uint4*>(tile) + i;
                const uint4 v = *w;
                *w = make_uint4(recode4<F>(v.x, ratio), recode4<F>(v.y, ratio), recode4<F>(v.z, ratio),
                                recode4<F>(v.w, ratio));
            }
        }
        __syncwarp();
    }
    if (lane == 0) *scale = pow2(x);
    const double inv = double(pow2(-x));
    for (int t = sub; t < n; t += kStep) {
        double r[8];
        load_rotated(at + t * stride, ch, p.interleaved, p.cos, p.sin, rotary, position + t, r);
        unsigned char* to = tile + (slot0 + t) * D;
        *reinterpret_cast<uint32_t*>(to + ch.i0) = encode4<F>(r, 0, inv);
        *reinterpret_cast<uint32_t*>(to + ch.i1) = encode4<F>(r, 4, inv);
    }
    if (__any_sync(0xffffffffu, odd) && lane == 0) raise_error(p.error, kErrValue);
}

// One CTA per packed row: it rotates the row's q, and the first row of each touched block
// writes the block's tiles.
template <class T, int F, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
    pdl_enter();
    __shared__ int s_seq;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x;
    if (tid == 0) s_seq = 0;
    __syncthreads();
    // the row's sequence: the number of sequences that end at or before it
    int before = 0;
    for (int i = tid; i < p.count; i += kThreads) before += p.row_offsets[i + 1] <= row;
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) atomicAdd(&s_seq, before);
    __syncthreads();
    const int seq = s_seq;
    if (seq >= p.count) return;  // behind the last sequence
    const int begin = p.row_offsets[seq], end = min(p.row_offsets[seq + 1], p.rows), start = p.starts[seq];
    const int64_t position = int64_t(start) + row - begin;
    if (row < begin || row >= end || start < 0 || position >= int64_t(p.table_stride) * p.cache.block_tokens ||
        (p.rotary_dim && position >= p.max_positions)) {
        if (tid == 0) raise_error(p.error, kErrBounds);
        return;
    }
    const int pos = int(position), bt = p.cache.block_tokens, slot = pos % bt;
    if (p.q) {
        const T* q = static_cast<const T*>(p.q) + row * p.q_stride;
        T* out = static_cast<T*>(p.q_out) + row * p.q_out_stride;
        for (int i = tid; i < p.heads * (D / 8); i += kThreads) {
            const int head = i / (D / 8), c = i % (D / 8);
            const Chunk ch = chunk_of(c, p.rotary_dim, p.interleaved);
            double r[8];
            load_rotated(q + head * D, ch, p.interleaved, p.cos, p.sin, p.rotary_dim, pos, r);
            store4(out + head * D + ch.i0, rounded(r[0], T{}), rounded(r[1], T{}), rounded(r[2], T{}), rounded(r[3], T{}));
            store4(out + head * D + ch.i1, rounded(r[4], T{}), rounded(r[5], T{}), rounded(r[6], T{}), rounded(r[7], T{}));
        }
    }
    if (row != begin && slot != 0) return;
    const int block = p.tables[int64_t(seq) * p.table_stride + pos / bt];
    int n = min(bt - slot, end - row);
    if (p.rotary_dim) n = min(n, p.max_positions - pos);  // rows past the tables report themselves
    if (unsigned(block) >= unsigned(p.cache.max_blocks)) {
        if (tid == 0) raise_error(p.error, kErrBounds);
        return;
    }
    for (int i = warp; i < 2 * p.cache.kv_heads; i += kThreads / 32) {
        const int head = i >> 1, part = i & 1;
        if (part == 0) {
            append_tile<T, F, D>(p, static_cast<const T*>(p.k) + row * p.k_stride, p.k_stride, head, 0, block, slot, n, pos, lane);
        } else {
            append_tile<T, F, D>(p, static_cast<const T*>(p.v) + row * p.v_stride, p.v_stride, head, 1, block, slot, n, pos, lane);
        }
    }
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    return dispatch(type, format, head_dim, [&](auto t, auto f, auto d) {
        return launch_pdl(append_kernel<decltype(t), decltype(f)::value, decltype(d)::value>, dim3(p.rows),
                          dim3(kThreads), 0, stream, p);
    });
}

}  // namespace kv8
}  // namespace mpb
