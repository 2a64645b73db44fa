// Entry points of the 8-bit paged K/V cache operators: argument checks, then one
// launch on the caller's stream. Nothing here allocates, copies or synchronises
// (mp_kv8_status alone synchronises).
#include <atomic>

#include "kv8.cuh"

namespace {

using namespace mpb;

std::atomic<unsigned> stall_next_ns{0};  // mp_kv8_inject_wait_timeout

int refuse(int code, const char* message) {
    set_last_error(message);
    return code;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const mp_kv8_cache* c) {
    if (!c || !c->pages || !c->scales) return refuse(MP_ERR_INVALID, "kv8: null cache");
    if (c->format != MP_KV8_INT8 && c->format != MP_KV8_E4M3) return refuse(MP_ERR_INVALID, "kv8: unknown format");
    if (c->kv_heads < 1 || c->kv_heads > 256 || c->max_blocks < 1)
        return refuse(MP_ERR_INVALID, "kv8: kv_heads or max_blocks out of range");
    if (c->head_dim != 64 && c->head_dim != 128) return refuse(MP_ERR_UNSUPPORTED, "kv8: head_dim is not 64 or 128");
    if (c->block_tokens < 16 || c->block_tokens > 256 || c->block_tokens % 16)
        return refuse(MP_ERR_UNSUPPORTED, "kv8: block_tokens is not a multiple of 16 up to 256");
    if (c->page_stride < int64_t(c->kv_heads) * 2 * c->block_tokens * c->head_dim || c->page_stride % 16)
        return refuse(MP_ERR_INVALID, "kv8: page_stride below a block's bytes or no multiple of 16");
    if (c->scale_stride < 2 * c->kv_heads || c->scale_stride % 2)
        return refuse(MP_ERR_INVALID, "kv8: scale_stride below 2 * kv_heads or odd");
    if (!aligned(c->pages, 16) || !aligned(c->scales, 8)) return refuse(MP_ERR_INVALID, "kv8: misaligned cache");
    return MP_OK;
}

int check_rows(const mp_kv8_cache* c, int type, int heads, int count, int table_stride) {
    if (type != MP_TYPE_F32 && type != MP_TYPE_BF16) return refuse(MP_ERR_INVALID, "kv8: unknown type");
    if (heads < 1 || heads > 1024 || heads % c->kv_heads || heads / c->kv_heads > 64)
        return refuse(MP_ERR_INVALID, "kv8: heads is not 1 to 64 times kv_heads, or above 1024");
    if (count < 1 || count > 65536 || table_stride < 1)
        return refuse(MP_ERR_INVALID, "kv8: count or table_stride out of range");
    if (int64_t(table_stride) * c->block_tokens > kv8::kMostTokens)
        return refuse(MP_ERR_INVALID, "kv8: a table of more than 2^26 tokens");
    return MP_OK;
}

// Rows of `width` values: 16-byte aligned base and stride, rows that do not overlap.
int check_buffer(const void* p, int64_t stride, int64_t width, int type) {
    const int64_t per = type == MP_TYPE_F32 ? 4 : 8;
    if (!p || !aligned(p, 16)) return refuse(MP_ERR_INVALID, "kv8: null or misaligned row buffer");
    if (stride < width || stride % per) return refuse(MP_ERR_INVALID, "kv8: row stride below the row or misaligned");
    return MP_OK;
}

int check_words(const void* p) {
    return p && aligned(p, 4) ? MP_OK : refuse(MP_ERR_INVALID, "kv8: null or misaligned metadata");
}

// Every pointer is memory of the current device (or managed): a host array or another
// device's buffer would fault in the kernel.
int check_device(std::initializer_list<const void*> pointers) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return refuse(MP_ERR_CUDA, "kv8: no usable current CUDA device");
    for (const void* p : pointers) {
        if (!p) continue;
        cudaPointerAttributes a{};
        const cudaError_t e = cudaPointerGetAttributes(&a, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return refuse(MP_ERR_CUDA, cudaGetErrorString(e));
        }
        if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != device))
            return refuse(MP_ERR_INVALID, "kv8: a pointer is not memory of the current device");
    }
    return MP_OK;
}

int finish(cudaError_t e) {
    if (e == cudaSuccess) return MP_OK;
    cudaGetLastError();
    return refuse(MP_ERR_CUDA, cudaGetErrorString(e));
}

kv8::Cache view(const mp_kv8_cache* c) {
    return {static_cast<unsigned char*>(c->pages), c->scales,       c->page_stride, c->scale_stride,
            c->kv_heads,                           c->block_tokens, c->max_blocks};
}

bool geometry(const mp_kv8_cache* c, int heads) {
    return c && c->kv_heads >= 1 && (c->head_dim == 64 || c->head_dim == 128) && heads >= 1 && heads % c->kv_heads == 0;
}

#define MPB_TRY(x)                  \
    do {                            \
        const int rc_ = (x);        \
        if (rc_ != MP_OK) return rc_; \
    } while (0)

}  // namespace

extern "C" int mp_kv8_append(const mp_kv8_cache* cache, const mp_kv8_append_args* a, uint32_t* device_error,
                             void* stream) {
    MPB_TRY(check_cache(cache));
    if (!a) return refuse(MP_ERR_INVALID, "kv8: null arguments");
    const int64_t d = cache->head_dim;
    MPB_TRY(check_rows(cache, a->type, a->heads, a->count, a->table_stride));
    if (a->rows < 0) return refuse(MP_ERR_INVALID, "kv8: negative rows");
    if (a->rotary_dim < 0 || a->rotary_dim > d || a->rotary_dim % 8)
        return refuse(MP_ERR_INVALID, "kv8: rotary_dim is not a multiple of 8 up to head_dim");
    if (a->rope_layout != MP_ROPE_HALF && a->rope_layout != MP_ROPE_INTERLEAVED)
        return refuse(MP_ERR_INVALID, "kv8: unknown rope_layout");
    if (a->rotary_dim && (!a->cos || !a->sin || !aligned(a->cos, 16) || !aligned(a->sin, 16) || a->max_positions < 1))
        return refuse(MP_ERR_INVALID, "kv8: null, misaligned or empty rotation tables");
    MPB_TRY(check_buffer(a->k, a->k_stride, cache->kv_heads * d, a->type));
    MPB_TRY(check_buffer(a->v, a->v_stride, cache->kv_heads * d, a->type));
    if (!a->q != !a->q_out) return refuse(MP_ERR_INVALID, "kv8: q without q_out or q_out without q");
    if (a->q) {
        MPB_TRY(check_buffer(a->q, a->q_stride, a->heads * d, a->type));
        MPB_TRY(check_buffer(a->q_out, a->q_out_stride, a->heads * d, a->type));
        if (a->q_out == a->q && a->q_out_stride != a->q_stride)
            return refuse(MP_ERR_INVALID, "kv8: q rotated in place with another row stride");
    }
    MPB_TRY(check_words(a->tables));
    MPB_TRY(check_words(a->row_offsets));
    MPB_TRY(check_words(a->starts));
    if (device_error) MPB_TRY(check_words(device_error));
    MPB_TRY(check_device({cache->pages, cache->scales, a->q, a->k, a->v, a->q_out, a->rotary_dim ? a->cos : nullptr,
                          a->rotary_dim ? a->sin : nullptr, a->tables, a->row_offsets, a->starts, device_error}));
    if (a->rows == 0) return MP_OK;
    kv8::AppendParams p{};
    p.cache = view(cache);
    p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
    p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride, p.q_out_stride = a->q_out_stride;
    p.cos = a->cos, p.sin = a->sin;
    p.tables = a->tables, p.row_offsets = a->row_offsets, p.starts = a->starts;
    p.heads = a->heads, p.rotary_dim = a->rotary_dim, p.interleaved = a->rope_layout == MP_ROPE_INTERLEAVED;
    p.max_positions = a->max_positions, p.table_stride = a->table_stride, p.count = a->count, p.rows = a->rows;
    p.error = device_error;
    return finish(kv8::launch_append(p, a->type, cache->format, cache->head_dim, static_cast<cudaStream_t>(stream)));
}

extern "C" size_t mp_kv8_decode_workspace(const mp_kv8_cache* cache, int32_t heads) {
    return geometry(cache, heads) ? kv8::decode_workspace(heads / cache->kv_heads, cache->head_dim) : 0;
}

extern "C" size_t mp_kv8_prefill_workspace(const mp_kv8_cache* cache, int32_t heads) {
    return geometry(cache, heads) ? kv8::prefill_workspace(heads / cache->kv_heads, cache->head_dim) : 0;
}

extern "C" int mp_kv8_attention_decode(const mp_kv8_cache* cache, const mp_kv8_decode_args* a, uint32_t* device_error,
                                       void* stream) {
    MPB_TRY(check_cache(cache));
    if (!a) return refuse(MP_ERR_INVALID, "kv8: null arguments");
    MPB_TRY(check_rows(cache, a->type, a->heads, a->count, a->table_stride));
    const int64_t width = int64_t(a->heads) * cache->head_dim;
    MPB_TRY(check_buffer(a->q, a->q_stride, width, a->type));
    MPB_TRY(check_buffer(a->out, a->out_stride, width, a->type));
    MPB_TRY(check_words(a->tables));
    MPB_TRY(check_words(a->lengths));
    if (device_error) MPB_TRY(check_words(device_error));
    if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < mp_kv8_decode_workspace(cache, a->heads))
        return refuse(MP_ERR_INVALID, "kv8: null, misaligned or short workspace");
    MPB_TRY(check_device({cache->pages, cache->scales, a->q, a->out, a->tables, a->lengths, a->workspace, device_error}));
    kv8::AttentionParams p{};
    p.cache = view(cache);
    p.q = a->q, p.out = a->out, p.q_stride = a->q_stride, p.out_stride = a->out_stride;
    p.tables = a->tables, p.lengths = a->lengths, p.workspace = a->workspace;
    p.heads = a->heads, p.table_stride = a->table_stride, p.count = a->count, p.rows = a->count;
    p.scale = a->scale;
    p.error = device_error;
    return finish(kv8::launch_decode(p, a->type, cache->format, cache->head_dim, static_cast<cudaStream_t>(stream)));
}

extern "C" int mp_kv8_attention_prefill(const mp_kv8_cache* cache, const mp_kv8_prefill_args* a,
                                        uint32_t* device_error, void* stream) {
    MPB_TRY(check_cache(cache));
    if (!a) return refuse(MP_ERR_INVALID, "kv8: null arguments");
    MPB_TRY(check_rows(cache, a->type, a->heads, a->count, a->table_stride));
    if (a->rows < 0) return refuse(MP_ERR_INVALID, "kv8: negative rows");
    const int64_t width = int64_t(a->heads) * cache->head_dim;
    MPB_TRY(check_buffer(a->q, a->q_stride, width, a->type));
    MPB_TRY(check_buffer(a->out, a->out_stride, width, a->type));
    MPB_TRY(check_words(a->tables));
    MPB_TRY(check_words(a->row_offsets));
    MPB_TRY(check_words(a->starts));
    if (device_error) MPB_TRY(check_words(device_error));
    if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < mp_kv8_prefill_workspace(cache, a->heads))
        return refuse(MP_ERR_INVALID, "kv8: null, misaligned or short workspace");
    MPB_TRY(check_device({cache->pages, cache->scales, a->q, a->out, a->tables, a->row_offsets, a->starts,
                          a->workspace, device_error}));
    if (a->rows == 0) return MP_OK;
    kv8::AttentionParams p{};
    p.cache = view(cache);
    p.q = a->q, p.out = a->out, p.q_stride = a->q_stride, p.out_stride = a->out_stride;
    p.tables = a->tables, p.row_offsets = a->row_offsets, p.starts = a->starts, p.workspace = a->workspace;
    p.heads = a->heads, p.table_stride = a->table_stride, p.count = a->count, p.rows = a->rows;
    p.scale = a->scale;
    p.error = device_error;
    p.stall_ns = stall_next_ns.exchange(0, std::memory_order_relaxed);
    return finish(kv8::launch_prefill(p, a->type, cache->format, cache->head_dim, static_cast<cudaStream_t>(stream)));
}

extern "C" int mp_kv8_inject_wait_timeout(int32_t wait_us) {
    if (wait_us < 1 || wait_us > 1000000) return refuse(MP_ERR_INVALID, "kv8: wait limit must be 1 us .. 1 s");
    stall_next_ns.store(unsigned(wait_us) * 1000u, std::memory_order_relaxed);
    return MP_OK;
}

extern "C" int mp_kv8_status(uint32_t* device_error, void* stream_ptr) {
    if (!device_error || !aligned(device_error, 4)) return refuse(MP_ERR_INVALID, "kv8: null or misaligned error word");
    MPB_TRY(check_device({device_error}));
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    unsigned bits = 0;
    cudaError_t e = cudaMemcpyAsync(&bits, device_error, sizeof(bits), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e == cudaSuccess && bits) e = cudaMemsetAsync(device_error, 0, sizeof(bits), stream);
    if (e != cudaSuccess) return finish(e);
    if (bits & kErrTimeout) return refuse(MP_ERR_TIMEOUT, "kv8: a wait expired");
    if (bits & kErrBounds) return refuse(MP_ERR_BOUNDS, "kv8: block id, metadata or position out of range");
    if (bits & kv8::kErrValue) return refuse(MP_ERR_NONFINITE, "kv8: value or block scale that cannot be quantised");
    return MP_OK;
}
