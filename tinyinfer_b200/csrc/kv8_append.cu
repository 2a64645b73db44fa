// mp_kv8_append: rotate q and k, quantise k and v, write the 8-bit pages (sm_100a).
//
// Rotation of a pair (a, b) at position p with c = cos[p][i], s = sin[p][i]: (a c - b s,
// b c + a s), the reference's rope_append step (miniprefix/src/backend/cuda/
// llama_runner.cu:20-32). A rotated q is one product and one fused multiply-add.
//
// A k code is the nearest multiple of the block's scale to the exact rotated value, so a
// value next to the border of two codes must not be rounded on the way. The FP32 value
// a c - (b s) is off by at most e = 2^-23 (|b s| + |value|), far below a code (|b s| is at most
// the rotated pair's length); where value - e and value + e have the same code, that is the
// code. Where not (one value in some 10^4) the lane computes its codes again in 64 bits, in
// which the products are exact; likewise for the scale, and for tiles with values outside the
// range in which e holds. (Everything in 64 bits measured 24 us for 8192 rows of 9 + 3 + 3 heads
// x 64 FP32, and 290 us for 20447 rows of 32 + 8 + 8 heads x 128 BF16: its conversions bound it.)
//
// A CTA takes up to 8 packed rows: its warps write the tiles of the blocks that begin among
// its rows (a tile's first appended row is in one CTA only), or all its threads rotate
// their q; one CTA does both, or two share the rows (launch_append). A tile is (block, kv head,
// K or V); its scale needs the largest magnitude of all its new tokens, so one warp takes it
// whole, 16 tokens (8 of head_dim 128) in registers at a time, twice: magnitude, then codes.
// Fewer rows per CTA when there are few (one for a decode step), so that all SMs take part.
//
// Measured with buffers that pass through L2: 8192 rows of 9 + 3 + 3 heads x 64 FP32 17.8 us (3.1
// TB/s; 15.4 where they stay in it), 20447 of 32 + 8 + 8 heads x 128 BF16 130 us (3.9 TB/s), 0.47
// and 0.59 of the copy rate: a warp's loads, magnitude and codes follow one another, and the 20
// warps of an SM hide part of that. Large blocks leave most warps without a tile: the 8192 rows
// take 31 us with blocks of 64 tokens and 87 with 256.
#include "kv8.cuh"

namespace mpb {
namespace kv8 {
namespace {

constexpr int kMaxRows = 8;  // rows of a CTA (16 and 4 were no faster)
constexpr float kHuge = 8.5e37f;  // 2^126: FP32 products and sums below it are finite

// A lane's eight values of one head row: two groups of four, at i0 and i1. Chunk c of
// the rotated dims holds four whole pairs; later chunks pass through.
struct Chunk {
    int i0, i1, pair;  // pair: index of the first of the four rotation pairs, -1: none
};
template <bool kInterleaved>
__device__ __forceinline__ Chunk chunk_of(int c, int rotary) {
    if (8 * c >= rotary) return {8 * c, 8 * c + 4, -1};
    return kInterleaved ? Chunk{8 * c, 8 * c + 4, 4 * c} : Chunk{4 * c, rotary / 2 + 4 * c, 4 * c};
}

// The chunk's eight values as they are in memory.
template <class T>
struct Raw {
    using Word = std::conditional_t<sizeof(T) == 4, float4, uint2>;  // four values
    Word a, b;
    __device__ __forceinline__ void load(const T* row, Chunk ch) {
        a = *reinterpret_cast<const Word*>(row + ch.i0);
        b = *reinterpret_cast<const Word*>(row + ch.i1);
    }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        widen4f(a, x);
        widen4f(b, x + 4);
    }
    static __device__ __forceinline__ void widen4f(float4 w, float* x) { x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w; }
    static __device__ __forceinline__ void widen4f(uint2 w, float* x) {
        x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xffff0000u);
        x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
};

// What a rotation reads: the tables' row of a position.
struct Angles {
    const float *cos, *sin;
    int half;
    __device__ __forceinline__ void load(int position, int pair, float (&c)[4], float (&s)[4]) const {
        const size_t at = size_t(position) * half + pair;
        load4(cos + at, c);
        load4(sin + at, s);
    }
};

// Rotates a chunk in FP32; returns the largest magnitude of its rounded products.
template <bool kInterleaved>
__device__ __forceinline__ float rotate(float (&x)[8], const float (&c)[4], const float (&s)[4]) {
    float cross = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float &a = x[kInterleaved ? 2 * i : i], &b = x[kInterleaved ? 2 * i + 1 : 4 + i];
        const float bs = __fmul_rn(b, s[i]), as = __fmul_rn(a, s[i]);
        cross = fmaxf(cross, fmaxf(fabsf(bs), fabsf(as)));
        a = __fmaf_rn(a, c[i], -bs);
        b = __fmaf_rn(b, c[i], as);
    }
    return cross;
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

// Codes of two values in units of the scale, in the low two bytes. INT8: adding 1.5 * 2^23
// rounds to an integer (ties to even) whose low byte is the code; |value| <= 127.5.
template <int F>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
    if constexpr (F == MP_KV8_INT8) {
        return __byte_perm(__float_as_uint(__fadd_rn(a, 12582912.f)), __float_as_uint(__fadd_rn(b, 12582912.f)), 0x0040) &
               0xffffu;
    } else {
        uint16_t h;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(b), "f"(a));
        return h;
    }
}
template <int F>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (F == MP_KV8_INT8) {
        const uint32_t x = __byte_perm(__float_as_uint(__fadd_rn(a, 12582912.f)), __float_as_uint(__fadd_rn(b, 12582912.f)), 0x0040);
        const uint32_t y = __byte_perm(__float_as_uint(__fadd_rn(c, 12582912.f)), __float_as_uint(__fadd_rn(d, 12582912.f)), 0x0040);
        return __byte_perm(x, y, 0x5410);
    } else {
        return encode2<F>(a, b) | encode2<F>(c, d) << 16;
    }
}

// Four held codes times `ratio` (a power of two below 1), rounded to codes again.
template <int F>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
    uint32_t lo, hi;
    widen4<F>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    return encode4<F>(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

// ---------------------------------------------------------------- in 64 bits
// One value of a row: dim `d`, rotated.
template <class T, bool kInterleaved>
__device__ double exact_value(const T* row, int d, const Angles& angles, int rotary, int position) {
    const double x = double(float(row[d]));
    if (d >= rotary) return x;
    const int half = rotary / 2;
    const int i = kInterleaved ? d / 2 : d % half;
    const bool second = kInterleaved ? d & 1 : d >= half;
    const int other = kInterleaved ? d ^ 1 : second ? d - half : d + half;
    const double y = double(float(row[other]));
    const double c = double(angles.cos[size_t(position) * half + i]), s = double(angles.sin[size_t(position) * half + i]);
    return second ? x * c + y * s : x * c - y * s;
}

// Its code; NaN is 0, infinity the largest. (A 64-bit value rounds to odd in 32 bits first, so
// that rounding those to a code is one rounding.)
template <int F>
__device__ uint32_t exact_code(double v, float inv) {
    if (isnan(v)) return 0;
    const double y = v * double(inv);
    if constexpr (F == MP_KV8_INT8) {
        return uint32_t(__double2int_rn(fmin(fmax(y, -127.0), 127.0)) & 255);
    } else {
        float f = __double2float_rz(y);
        if (double(f) != y) f = __int_as_float(__float_as_int(f) | 1);
        return encode2<F>(f, 0.f) & 255u;
    }
}

// A chunk's codes: those at i0 and at i1.
template <class T, int F, bool kInterleaved>
__device__ __noinline__ uint2 exact_codes(const T* row, int i0, int i1, Angles angles, int rotary, int position, float inv) {
    uint32_t w[2] = {0, 0};
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        const int d = i < 4 ? i0 + i : i1 + i - 4;
        const uint32_t c = exact_code<F>(exact_value<T, kInterleaved>(row, d, angles, rotary, position), inv) << (8 * (i & 3));
        if (i < 4) {
            w[0] |= c;
        } else {
            w[1] |= c;
        }
    }
    return make_uint2(w[0], w[1]);
}

// A warp's tile: the largest finite magnitude, rounded to 32 bits; *odd: some value is not finite.
template <class T, bool kInterleaved>
__device__ __noinline__ float exact_largest(const T* at, int64_t stride, int n, int dims, Angles angles, int rotary,
                                            int position, int lane, bool* odd) {
    float amax = 0.f;
    bool bad = false;
#pragma unroll 1
    for (int i = lane; i < n * dims; i += 32) {
        const int t = i / dims;
        const float f = fabsf(__double2float_rn(exact_value<T, kInterleaved>(at + t * stride, i % dims, angles, rotary, position + t)));
        const bool finite = f <= 3.402823466e38f;
        bad |= !finite;
        amax = finite ? fmaxf(amax, f) : amax;
    }
    *odd = __any_sync(0xffffffffu, bad);
    return warp_max(amax);
}

// ---------------------------------------------------------------- a tile, by one warp
template <class T, int F, int D, bool kInterleaved>
__device__ __forceinline__ void append_tile(const AppendParams& p, const T* rows, int64_t stride, int head, int part,
                                            const int32_t* entry, int slot0, int n, int position, int lane) {
    constexpr int kLanes = D / 8;        // lanes of one token
    constexpr int kStep = 32 / kLanes;   // tokens a warp reads at once
    constexpr int kSteps = 4, kUnitTokens = kSteps * kStep;  // a lane's tokens at a time, and the warp's
    const int sub = lane / kLanes, rotary = part ? 0 : p.rotary_dim;
    const Angles angles{p.cos, p.sin, rotary / 2};
    const Chunk ch = chunk_of<kInterleaved>(lane % kLanes, rotary);
    const T* at = rows + head * D;
    // a lane's values of kSteps tokens, rotated; what any of a token's may be off by (0: they are exact)
    float x[kSteps][8], e[kSteps];
    Raw<T> raw[kSteps];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int t = first + i * kStep + sub;
            raw[i] = {};
            if (t < n) raw[i].load(at + t * stride, ch);
        }
    };
    auto turn = [&](int first) {
        if (ch.pair >= 0) {
            float c[kSteps][4], s[kSteps][4];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) angles.load(position + min(first + i * kStep + sub, n - 1), ch.pair, c[i], s[i]);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                raw[i].widen(x[i]);
                e[i] = rotate<kInterleaved>(x[i], c[i], s[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) raw[i].widen(x[i]), e[i] = 0.f;
        }
    };
    load(0);
    const int block = *entry;  // in flight with the values
    // bounds of the largest magnitude; `sum` becomes NaN if a value is not finite
    float most = 0.f, least = 0.f, sum = 0.f;
    for (int first = 0; first < n; first += kUnitTokens) {
        if (first) load(first);
        turn(first);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j])), sum = fmaf(x[i][j], 0.f, sum);
            if (ch.pair >= 0) e[i] = (e[i] + top) * 1.1920929e-7f;
            most = fmaxf(most, top + e[i]);
            least = fmaxf(least, top - e[i]);
        }
    }
    const bool wide = __any_sync(0xffffffffu, !(most < kHuge) || isnan(sum));  // e does not hold, or not finite
    most = warp_max(most), least = warp_max(least);
    if (unsigned(block) >= unsigned(p.cache.max_blocks)) {
        if (lane == 0) raise_error(p.error, kErrBounds);
        return;
    }
    bool odd = false;
    int power = scale_exponent<F>(least);
    if (wide || power != scale_exponent<F>(most))
        power = scale_exponent<F>(exact_largest<T, kInterleaved>(at, stride, n, D, angles, rotary, position, lane, &odd));
    float* scale = p.cache.scales + int64_t(block) * p.cache.scale_stride + head * 2 + part;
    unsigned char* tile = p.cache.pages + tile_offset(p.cache, block, head, part, D);
    if (slot0 > 0) {
        const float held = *scale;
        const int bits = __float_as_int(held), e = (bits >> 23) - 127;
        if ((bits & 0x807fffff) != 0 || e < -126 || e > 127) {
            odd = true;  // not a power of two: the held codes stay as they are under the new scale
        } else if (e >= power) {
            power = e;
        } else {
            const float ratio = e - power < -126 ? 0.f : pow2(e - power);
            for (int i = lane; i < slot0 * D / 16; i += 32) {
                uint4* w = reinterpret_cast<uint4*>(tile) + i;
                const uint4 v = *w;
                *w = make_uint4(recode4<F>(v.x, ratio), recode4<F>(v.y, ratio), recode4<F>(v.z, ratio),
                                recode4<F>(v.w, ratio));
            }
        }
        __syncwarp();
    }
    if (lane == 0) *scale = pow2(power);
    // a held scale may be 2^127: its inverse is subnormal (a new scale is at most 2^122)
    const float inv = power == 127 ? 5.877471754e-39f : pow2(-power);
    for (int first = 0; first < n; first += kUnitTokens) {
        if (n > kUnitTokens) {  // else still there
            load(first);
            turn(first);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int t = first + i * kStep + sub;
            if (t >= n) continue;
            uint32_t w[2];
            bool near = wide;  // a border of codes lies within what a value may be off by
            if (ch.pair < 0) {
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    w[j / 4] = encode4<F>(x[i][j] * inv, x[i][j + 1] * inv, x[i][j + 2] * inv, x[i][j + 3] * inv);
            } else {
                if (n > kUnitTokens) {
                    float top = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j]));
                    e[i] = (e[i] + top) * 1.1920929e-7f;
                }
                const float d = fmaf(e[i], inv, 9.094947e-13f);  // 2^-40: products that lost bits below FP32's exponents
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    const float* v = x[i] + j;
                    w[j / 4] = encode4<F>(fmaf(v[0], inv, -d), fmaf(v[1], inv, -d), fmaf(v[2], inv, -d), fmaf(v[3], inv, -d));
                    near |= w[j / 4] != encode4<F>(fmaf(v[0], inv, d), fmaf(v[1], inv, d), fmaf(v[2], inv, d), fmaf(v[3], inv, d));
                }
            }
            if (near) {
                const uint2 exact = exact_codes<T, F, kInterleaved>(at + t * stride, ch.i0, ch.i1, angles, rotary, position + t, inv);
                w[0] = exact.x, w[1] = exact.y;
            }
            unsigned char* to = tile + (slot0 + t) * D;
            *reinterpret_cast<uint32_t*>(to + ch.i0) = w[0];
            *reinterpret_cast<uint32_t*>(to + ch.i1) = w[1];
        }
    }
    if (odd && lane == 0) raise_error(p.error, kErrValue);
}

// A packed row's place: its sequence (-1: behind the last, or of one that is out of range) and position.
struct Place {
    int seq, position, end;  // end: the sequence's last row + 1
};

// Positions that a sequence may have: those of its table (at most kMostTokens) and of the rotation tables.
__device__ __forceinline__ int position_limit(const AppendParams& p) {
    const int tokens = p.table_stride * p.cache.block_tokens;
    return p.rotary_dim ? min(tokens, p.max_positions) : tokens;
}

// By one warp, a row per lane from `row0` on (rows <= 32): a row's sequence is the first that
// ends behind it. With sequences of one length it is known for row0; else it is found 32
// ways at a time. From there on step by step.
__device__ __forceinline__ Place find_rows(const AppendParams& p, int row0, int rows, int lane) {
    int low = int(int64_t(row0) * p.count / p.rows);
    const int guess = low, start_there = p.starts[low];
    if (p.row_offsets[low] > row0 || p.row_offsets[low + 1] <= row0) {
        low = 0;
        int high = p.count;
        while (high - low > 32) {
            const int step = (high - low + 31) / 32, i = low + (lane + 1) * step - 1;
            const int k = __popc(__ballot_sync(0xffffffffu, i < high && p.row_offsets[i + 1] <= row0));
            low += k * step;
            high = min(high, low + step);
        }
        low += __popc(__ballot_sync(0xffffffffu, low + lane < high && p.row_offsets[low + lane + 1] <= row0));
    }
    const int row = row0 + lane;
    if (lane >= rows) return {-1, 0, 0};
    int end = 0;
    while (low < p.count && (end = p.row_offsets[low + 1]) <= row) ++low;
    if (low >= p.count) return {-1, 0, 0};
    const int begin = p.row_offsets[low], start = low == guess ? start_there : p.starts[low];
    if (row < begin || checked_rows(begin, end, start, p.rows, position_limit(p), 1, nullptr) == 0) return {-1, 0, 0};
    return {low, start + row - begin, end};
}

template <class T, int F, int D, bool kInterleaved, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 5 : 2) append_kernel(const AppendParams p, int rows_each, uint32_t per_row_inverse) {
    constexpr int kChunks = D / 8;
    __shared__ Place places[kMaxRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_enter();
    const int row0 = blockIdx.x * rows_each, rows = min(rows_each, p.rows - row0);
    if (warp == 0) {
        const Place at = find_rows(p, row0, rows, lane);
        if (lane < rows) places[lane] = at;
    }
    __syncthreads();
    // ---- tiles of the blocks whose first appended row is here
    const int bt = p.cache.block_tokens, tiles = 2 * p.cache.kv_heads;
    int turn = warp;  // tiles go round the warps
    for (int i = 0; i < (blockIdx.y == 0 ? rows : 0); ++i) {
        const Place at = places[i];
        const int slot = at.position % bt;
        if (at.seq < 0) continue;
        if (slot && row0 + i != p.row_offsets[at.seq]) continue;
        const int row = row0 + i;
        const int32_t* entry = p.tables + int64_t(at.seq) * p.table_stride + at.position / bt;
        const int n = min(bt - slot, at.end - row);
        for (; turn < tiles; turn += kThreads / 32) {
            const int head = turn >> 1, part = turn & 1;
            const T* x = static_cast<const T*>(part ? p.v : p.k);
            const int64_t stride = part ? p.v_stride : p.k_stride;
            append_tile<T, F, D, kInterleaved>(p, x + row * stride, stride, head, part, entry, slot, n, at.position, lane);
        }
        turn -= tiles;
    }
    // ---- sequences that are out of range report themselves (here: before the tiles, beside the search for
    // the rows, this cost 8192 rows of 32 / 8 heads x 128 FP32 30 %)
    for (int i = blockIdx.x * kThreads + tid; blockIdx.y == 0 && i < p.count; i += gridDim.x * kThreads)
        checked_rows(p.row_offsets[i], p.row_offsets[i + 1], p.starts[i], p.rows, position_limit(p), 1, p.error);
    // ---- q: a chunk of a head of a row per thread, kFly of them in flight
    if (!p.q || blockIdx.y + 1 != gridDim.y) return;
    constexpr int kFly = kThreads == 128 ? 8 : 4;  // 20447 rows: 136 us with 4, 128 with 8; 256 single rows: 5.1 and 5.4
    const int per_row = p.heads * kChunks, total = rows * per_row;
    const Chunk ch = chunk_of<kInterleaved>(tid % kChunks, p.rotary_dim);  // kThreads is a multiple of kChunks
    const Angles angles{p.cos, p.sin, p.rotary_dim / 2};
    for (int first = tid; first < total; first += kFly * kThreads) {
        Raw<T> raw[kFly];
        int row[kFly], head[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            const int x = first + i * kThreads;
            row[i] = x < total ? int(__umulhi(x, per_row_inverse)) : 0;
            head[i] = (x - row[i] * per_row) / kChunks;
            if (x >= total || places[row[i]].seq < 0) {
                row[i] = -1;
            } else {
                raw[i].load(static_cast<const T*>(p.q) + (row0 + row[i]) * p.q_stride + head[i] * D, ch);
            }
        }
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            if (row[i] < 0) continue;
            float x[8];
            raw[i].widen(x);
            if (ch.pair >= 0) {
                float c[4], s[4];
                angles.load(places[row[i]].position, ch.pair, c, s);
                rotate<kInterleaved>(x, c, s);
            }
            T* to = static_cast<T*>(p.q_out) + (row0 + row[i]) * p.q_out_stride + head[i] * D;
            store4(to + ch.i0, x[0], x[1], x[2], x[3]);
            store4(to + ch.i1, x[4], x[5], x[6], x[7]);
        }
    }
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, int type, int format, int head_dim, cudaStream_t stream) {
    return dispatch(type, format, head_dim, [&](auto t, auto f, auto d) {
        const int each = std::clamp(p.rows / (2 * kCtas), 1, kMaxRows);
        using T = decltype(t);
        constexpr int kFormat = decltype(f)::value, kDim = decltype(d)::value;
        // x / per_row = high half of x * inverse while x * per_row < 2^32: x < 8 * per_row, per_row <= 2^14
        const uint32_t per_row = p.heads * (kDim / 8), inverse = uint32_t(((uint64_t(1) << 32) + per_row - 1) / per_row);
        // A row alone: 8 warps, so that its tiles are written side by side (5 rows, 256 rows: 4.1 and 5.1 us,
        // 5.3 and 5.9 with 4 warps). More rows: 4 warps, of which more CTAs overlap (8192 rows of FP32:
        // 17 us, 20 with 8 warps). The tiles' CTAs come before the queries' (of which more bytes are in
        // flight): 8192 rows 15.0 us against 16.7 with one CTA for both (17.7 in turn, 17.5 queries
        // first), 20447 rows of BF16 128 against 157, 5 rows 3.5 against 3.9. Single rows that fill
        // the SMs without are not split: 256 rows 5.1 us, 5.6 split.
        const int parts = p.q && (each > 1 || 2 * p.rows <= kCtas) ? 2 : 1;
        auto launch = [&](auto kernel, int threads) {
            return launch_pdl(kernel, dim3((p.rows + each - 1) / each, parts), dim3(threads), 0, stream, p, each, inverse);
        };
        if (each == 1)
            return p.interleaved ? launch(append_kernel<T, kFormat, kDim, true, 256>, 256)
                                 : launch(append_kernel<T, kFormat, kDim, false, 256>, 256);
        return p.interleaved ? launch(append_kernel<T, kFormat, kDim, true, 128>, 128)
                             : launch(append_kernel<T, kFormat, kDim, false, 128>, 128);
    });
}

}  // namespace kv8
}  // namespace mpb
