// Shared pieces of the 8-bit paged K/V cache operators (kv8_append.cu, kv8_decode.cu,
// kv8_prefill.cu): the cache view, code conversions and the checks of device-side
// metadata. The layout is mp_kv8_cache's (miniprefix_b200.h): a block holds, per kv
// head, a K tile and a V tile of [block_tokens][head_dim] bytes, each with one scale.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "miniprefix_b200.h"

namespace mpb {
namespace kv8 {

constexpr int kCtas = 148;            // one per SM
constexpr int kPackedItems = kCtas;   // items up to which a prefill goes row by row (kv8_prefill.cu)
constexpr int kCounterBytes = kCtas * 2 * 4 + 96;  // of the attentions' workspaces: zero between calls; partials follow
// Limits that keep a plan's 32-bit indexes in range: tokens of a table (checked by the host), and
// units of a CTA's run (checked by the device: minutes of work).
constexpr int64_t kMostTokens = int64_t(1) << 26, kMostUnits = int64_t(1) << 30;
constexpr unsigned kErrValue = 4u;  // error word bit: a value (or a held block's scale) that cannot be quantised

struct Cache {
    unsigned char* pages;
    float* scales;
    int64_t page_stride, scale_stride;
    int kv_heads, block_tokens, max_blocks;
};

struct AppendParams {
    Cache cache;
    const void *q, *k, *v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const float *cos, *sin;
    const int32_t *tables, *row_offsets, *starts;
    int heads, rotary_dim, interleaved, max_positions, table_stride, count, rows;
    unsigned* error;
};

struct AttentionParams {
    Cache cache;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int32_t* tables;
    const int32_t* lengths;      // decode
    const int32_t* row_offsets;  // prefill
    const int32_t* starts;       // prefill
    void* workspace;
    int heads, table_stride, count, rows;
    int sequences;  // launch_packed: of the prefill; count is its rows
    float scale;
    unsigned* error;
    unsigned stall_ns;  // failure-path tests: the prefill kernel's V tiles never come, and its waits end after this (0: none)
};

cudaError_t launch_append(const AppendParams& p, int type, int format, int head_dim, cudaStream_t stream);
cudaError_t launch_decode(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream);
cudaError_t launch_prefill(const AttentionParams& p, int type, int format, int head_dim, cudaStream_t stream);
// Prefill with at most kPackedItems (row, kv head, 8 query heads) items, row by row.
cudaError_t launch_packed(AttentionParams p, int type, int format, int head_dim, cudaStream_t stream);
size_t decode_workspace(int group, int head_dim);
size_t prefill_workspace(int group, int head_dim);

// Calls f with compile-time (type, format, head_dim); the arguments were checked.
template <class F>
cudaError_t dispatch(int type, int format, int head_dim, F f) {
    auto by_dim = [&](auto t, auto fmt) {
        return head_dim == 64 ? f(t, fmt, std::integral_constant<int, 64>{}) : f(t, fmt, std::integral_constant<int, 128>{});
    };
    auto by_format = [&](auto t) {
        return format == MP_KV8_INT8 ? by_dim(t, std::integral_constant<int, MP_KV8_INT8>{})
                                     : by_dim(t, std::integral_constant<int, MP_KV8_E4M3>{});
    };
    return type == MP_TYPE_F32 ? by_format(float{}) : by_format(__nv_bfloat16{});
}

// Position of 16-byte chunk `chunk` of token row `row` in a swizzled tile in shared memory.
template <int D>
__device__ __forceinline__ int swizzled(int row, int chunk) {
    return chunk ^ (D == 128 ? row & 7 : (row >> 1) & 3);
}

// Byte offset of the K (part 0) or V (part 1) tile of (block, kv head).
__device__ __forceinline__ int64_t tile_offset(const Cache& c, int block, int head, int part, int head_dim) {
    return int64_t(block) * c.page_stride + int64_t(head * 2 + part) * (c.block_tokens * head_dim);
}

// Block id of `page` in a table row; an id or page out of range sets the bounds bit
// and gives block 0, so that no access leaves the cache.
__device__ __forceinline__ int checked_id(const Cache& c, int b, unsigned* error) {
    if (unsigned(b) >= unsigned(c.max_blocks)) {
        raise_error(error, kErrBounds);
        return 0;
    }
    return b;
}
__device__ __forceinline__ int block_id(const Cache& c, const int32_t* table, int table_stride, int page,
                                        unsigned* error) {
    return checked_id(c, page < table_stride ? table[page] : -1, error);
}

// Rows of a sequence at row_offsets begin .. end of a call with `rows` packed ones, 0 if its metadata is out
// of range: offsets that fall or leave the call's rows, or positions past the `pages` times `tokens` there are.
__device__ __forceinline__ int checked_rows(int begin, int end, int start, int rows, int pages, int tokens, unsigned* error) {
    if (begin < 0 || end < begin || end > rows || (end > begin && start < 0) ||
        int64_t(start) + (end - begin) > int64_t(pages) * tokens) {
        if (end != begin) raise_error(error, kErrBounds);
        return 0;
    }
    return end - begin;
}

// Rows of a prefill's sequence i.
__device__ __forceinline__ int sequence_rows(const AttentionParams& p, int i, int& begin, int& start) {
    begin = p.row_offsets[i], start = p.starts[i];
    return checked_rows(begin, p.row_offsets[i + 1], start, p.rows, p.table_stride, p.cache.block_tokens, p.error);
}

// 2^x as a float, x in -126 .. 127.
__device__ __forceinline__ float pow2(int x) { return __int_as_float((x + 127) << 23); }

// ---------------------------------------------------------------- codes -> FP16 (exact)
// Four codes of one 32-bit word as two half2 registers (codes 0, 1 and 2, 3).
template <int F>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (F == MP_KV8_INT8) {
        // byte b + 128 under exponent byte 0x64 is the half 1024 + 128 + b: subtract 1152
        const uint32_t u = w ^ 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
        lo = *reinterpret_cast<uint32_t*>(&x);
        hi = *reinterpret_cast<uint32_t*>(&y);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// The same for a word of codes a0 a1 b0 b1 (two dims of tokens a and b): (a0, b0), (a1, b1).
template <int F>
__device__ __forceinline__ void widen_pairs(uint32_t w, uint32_t& first, uint32_t& second) {
    if constexpr (F == MP_KV8_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4240), b = __byte_perm(u, 0x64646464u, 0x4341);
        __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
        first = *reinterpret_cast<uint32_t*>(&x);
        second = *reinterpret_cast<uint32_t*>(&y);
    } else {
        widen4<F>(__byte_perm(w, 0, 0x3120), first, second);
    }
}

// FP16 halves of two values, packed: hi = fp16(x), lo = fp16(x - hi). Callers scale
// their values so that the largest are near 2^14: lo then keeps 11 bits of its own down
// to values 2^-26 of the largest, and hi + lo is x within 2^-22 |x|.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 2^x by the hardware approximation (relative error 2^-22; -inf gives 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Power-of-two factor that brings a row with largest magnitude `amax` into [2^14, 2^15)
// (near FP16's top, see split_pair), and its inverse. Rows below 2^-112 stay smaller.
__device__ __forceinline__ void row_factor(float amax, float& factor, float& inverse) {
    const int e = max((__float_as_int(amax) >> 23) & 255, 15);
    factor = __int_as_float((268 - e) << 23);
    inverse = __int_as_float((e - 14) << 23);
}

// D (16 x 8, FP32) += A (16 x 16) B (16 x 8), FP16 operands (warp-level tensor op).
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices of 16-bit elements from shared memory, transposed: lane l gives
// the address of row l % 8 of matrix l / 8. Volatile, so that it stays behind the wait for
// the copy that wrote the rows.
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address));
}

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
    __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
}

}  // namespace kv8
}  // namespace mpb
