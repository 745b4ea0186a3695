// int8_abi.cpp -- the extern "C" surface of the 8-bit serving operators (include/evelyn.h):
// checks of the arguments, the device they run on, the launches.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <new>

#include "engine.hpp"
#include "int8.h"

using namespace evl;

namespace {

template <class F> evl_status guarded(F&& f) {
    try {
        f();
        return EVL_OK;
    } catch (const Error& e) {
        set_last_error(e.msg);
        return e.code;
    } catch (const std::bad_alloc&) {
        set_last_error("out of host memory");
        return EVL_ERR_OUT_OF_MEMORY;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return EVL_ERR_IO;
    }
}

void require(bool ok, const char* msg) {
    if (!ok) raise(EVL_ERR_INVALID_INPUT, msg);
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

uint64_t elem_bytes(uint32_t type) {
    if (type == GGML_F32) return 4;
    if (type != GGML_F16 && type != GGML_BF16)
        raise(EVL_ERR_UNSUPPORTED, "activation type must be F32 (0), F16 (1) or BF16 (30)");
    return 2;
}

// Runs on the device that holds p; the caller's current device comes back afterwards.
struct OnDeviceOf {
    int dev = 0, prev = 0;
    explicit OnDeviceOf(const void* p) {
        cudaPointerAttributes at;
        cuda_check(cudaPointerGetAttributes(&at, p), "pointer attributes");
        require(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, "not a device pointer");
        dev = at.device;
        cuda_check(cudaGetDevice(&prev), "cudaGetDevice");
        if (prev != dev) cuda_check(cudaSetDevice(dev), "cudaSetDevice");
    }
    ~OnDeviceOf() {
        if (prev != dev) cudaSetDevice(prev);
    }
    OnDeviceOf(const OnDeviceOf&) = delete;
};

int sm_count(int dev) {
    static std::atomic<int> known[64];
    if (dev < 0 || dev >= 64) raise(EVL_ERR_UNSUPPORTED, "device index beyond 63");
    int n = known[dev].load();
    if (!n) {
        cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "device attribute");
        known[dev] = n;
    }
    return n;
}

Kv8Cache cache_of(const evl_kv8_cache* c) {
    require(c, "null cache");
    require(c->struct_size == sizeof(evl_kv8_cache), "evl_kv8_cache: struct_size is not this library's");
    require(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head_dim must be 64, 128 or 256");
    require(c->page_size == 16 || c->page_size == 32 || c->page_size == 64, "page_size must be 16, 32 or 64");
    require(c->kv_heads >= 1 && c->kv_heads <= 1024, "kv_heads must be 1..1024");
    require(c->n_pages <= 0x7fffffffu, "too many pages");
    const uint64_t codes = (uint64_t)c->kv_heads * c->page_size * c->head_dim;
    const uint64_t scales = (uint64_t)c->kv_heads * (c->page_size / 16);
    require(c->page_stride >= codes && c->page_stride % 16 == 0 && c->page_stride <= (1ull << 40),
            "page_stride must be a multiple of 16 bytes that holds a page");
    require(c->scale_stride >= scales && c->scale_stride <= (1ull << 40), "scale_stride must hold a page's scales");
    Kv8Cache r;
    r.kv_heads = c->kv_heads;
    r.head_dim = c->head_dim;
    r.page_size = c->page_size;
    r.n_pages = c->n_pages;
    r.k = c->d_k;
    r.v = c->d_v;
    r.ks = c->d_k_scales;
    r.vs = c->d_v_scales;
    r.page_stride = c->page_stride;
    r.scale_stride = c->scale_stride;
    return r;
}

void check_pages(const Kv8Cache& c) {
    require(c.k && c.v && c.ks && c.vs, "null cache buffer");
    require(aligned(c.k, 16) && aligned(c.v, 16), "code buffers must be 16-byte aligned");
    require(aligned(c.ks, 4) && aligned(c.vs, 4), "scale buffers must be 4-byte aligned");
}

Kv8Batch batch_of(const evl_kv8_batch* b) {
    require(b, "null batch");
    require(b->struct_size == sizeof(evl_kv8_batch), "evl_kv8_batch: struct_size is not this library's");
    require(b->n_seqs <= 65535, "at most 65535 sequences");
    require(b->total <= 0x3fffffffu, "too many tokens");
    require(b->max_len <= 0x3fffffffu, "max_len is too large");
    require(b->max_new >= 1 || !b->total || !b->n_seqs, "max_new must be at least 1");
    Kv8Batch r;
    r.n_seqs = b->n_seqs;
    r.total = b->total;
    r.max_new = std::min(b->max_new, b->total);
    r.max_len = b->max_len;
    r.table_stride = b->table_stride;
    r.table = b->d_page_table;
    r.cu = b->d_cu;
    r.len = b->d_len;
    return r;
}

void check_lists(const Kv8Batch& b) {
    require(b.table && b.cu && b.len, "null page table, cu or len");
    require(aligned(b.table, 4) && aligned(b.cu, 4) && aligned(b.len, 4), "page table, cu and len must be 4-byte aligned");
}

// Rows of activations that the kernels read or write in wide pieces.
void check_rows(const void* p, uint64_t stride, uint64_t width, uint64_t es, const char* what) {
    const std::string w(what);
    if (!p) raise(EVL_ERR_INVALID_INPUT, "null " + w);
    if (!aligned(p, 16) || (stride * es) % 16) raise(EVL_ERR_INVALID_INPUT, w + " must be 16-byte aligned, its stride a multiple of 16 bytes");
    if (stride < width || stride > (1ull << 40)) raise(EVL_ERR_INVALID_INPUT, w + ": the stride does not hold a token's heads");
}

// Whether two blocks of rows [rows][width], `stride` bytes apart in both (a single row has none), share memory.
bool share_memory(const void* a, const void* b, uint64_t rows, uint64_t width, uint64_t stride) {
    const uint64_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b), d = p < q ? q - p : p - q;
    if (d >= (rows - 1) * stride + width) return false;
    return rows == 1 || d % stride < width || stride - d % stride < width;
}

}  // namespace

extern "C" {

evl_status evl_i8_quantize_rows(uint32_t type, const void* d_x, uint64_t x_stride, uint32_t rows, uint32_t cols,
                                int8_t* d_codes, uint64_t code_stride, float* d_scales, void* stream) {
    return guarded([&] {
        const uint64_t es = elem_bytes(type);
        require(cols >= 1, "cols must be at least 1");
        require(rows <= 0x7fffffffu && cols <= 0x7fffffffu, "rows and cols must be below 2^31");
        if (!rows) return;
        require(d_x && d_codes && d_scales, "null argument");
        require(aligned(d_x, es) && aligned(d_scales, 4), "buffers must be aligned to their elements");
        require(x_stride >= cols && code_stride >= cols && x_stride <= (1ull << 40) && code_stride <= (1ull << 40),
                "strides must hold a row");
        OnDeviceOf on(d_x);
        QuantRowsArgs a;
        a.x = d_x;
        a.type = type;
        a.x_stride = x_stride;
        a.rows = rows;
        a.cols = cols;
        a.codes = d_codes;
        a.code_stride = code_stride;
        a.scales = d_scales;
        cuda_check(launch_quantize_rows(a, sm_count(on.dev), static_cast<cudaStream_t>(stream)), "quantize rows");
    });
}

evl_status evl_i8_matmul(const int8_t* d_x, uint64_t x_stride, const float* d_x_scales, uint32_t rows,
                         const int8_t* d_w, uint64_t w_stride, const float* d_w_scales, uint32_t out, uint32_t cols,
                         uint32_t type, const void* d_add, uint64_t add_stride, void* d_y, uint64_t y_stride,
                         int32_t* d_err, void* stream) {
    return guarded([&] {
        const uint64_t es = elem_bytes(type);
        require(cols >= 1 && cols <= 131071, "cols must be 1..131071");
        require(rows <= 0x3fffffffu && out <= 0x3fffffffu, "rows and out must be below 2^30");
        if (!rows || !out) return;
        require(d_x && d_x_scales && d_w && d_w_scales && d_y, "null argument");
        require(aligned(d_x, 16) && aligned(d_w, 16), "x and w must be 16-byte aligned");
        require(x_stride >= cols && w_stride >= cols && x_stride % 16 == 0 && w_stride % 16 == 0 &&
                    x_stride < (1ull << 40) && w_stride < (1ull << 40),
                "strides of x and w must be multiples of 16 bytes that hold a row");
        require(aligned(d_x_scales, 4) && aligned(d_w_scales, 4) && aligned(d_y, es) && aligned(d_err, 4) &&
                    (!d_add || aligned(d_add, es)),
                "buffers must be aligned to their elements");
        require(y_stride >= out && y_stride <= (1ull << 40) && (!d_add || (add_stride >= out && add_stride <= (1ull << 40))),
                "strides of y and add must hold a row");
        require(d_add != d_y || add_stride == y_stride, "add in place needs the stride of y");
        // (an output is written as soon as its own addition is read; blocks of different strides are not looked into)
        require(!d_add || d_add == d_y || (rows > 1 && add_stride != y_stride) ||
                    !share_memory(d_add, d_y, rows, out * es, y_stride * es),
                "add may be y, but must not overlap it otherwise");
        OnDeviceOf on(d_x);
        I8GemmArgs a;
        a.x = d_x;
        a.x_stride = x_stride;
        a.xs = d_x_scales;
        a.w = d_w;
        a.w_stride = w_stride;
        a.ws = d_w_scales;
        a.rows = rows;
        a.out = out;
        a.cols = cols;
        a.type = type;
        a.add = d_add;
        a.add_stride = add_stride;
        a.y = d_y;
        a.y_stride = y_stride;
        a.err = d_err;
        cuda_check(launch_i8_gemm(a, sm_count(on.dev), static_cast<cudaStream_t>(stream)), "8-bit matmul");
    });
}

// Not part of the public surface: how evl_i8_matmul cuts a product on the current device, so that the tests can
// see that their shapes reach every kernel (the rule is a fitted estimate).
evl_status evl_internal_i8_cut(uint32_t rows, uint32_t out, uint32_t cols, uint32_t type, uint32_t add, uint32_t* tokens,
                               uint32_t* split) {
    return guarded([&] {
        elem_bytes(type);
        require(rows && out && cols && tokens && split, "null argument");
        int dev = 0;
        cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
        I8GemmArgs a;
        a.rows = rows;
        a.out = out;
        a.cols = cols;
        a.type = type;
        a.add = add ? tokens : nullptr;  // (only whether there is one)
        i8_gemm_cut(a, sm_count(dev), *tokens, *split);
    });
}

evl_status evl_kv8_append(const evl_kv8_cache* cache, const evl_kv8_batch* batch, const evl_kv8_prep* prep,
                          uint32_t type, const void* d_k, uint64_t k_stride, const void* d_v, uint64_t v_stride,
                          const void* d_q, uint64_t q_stride, uint32_t heads, void* d_q_out, uint64_t q_out_stride,
                          int32_t* d_err, void* stream) {
    return guarded([&] {
        const uint64_t es = elem_bytes(type);
        Kv8AppendArgs a;
        a.c = cache_of(cache);
        a.b = batch_of(batch);
        a.type = type;
        if (prep) {
            require(prep->struct_size == sizeof(evl_kv8_prep), "evl_kv8_prep: struct_size is not this library's");
            if (prep->d_rope) {
                require(prep->rope_dim >= 4 && prep->rope_dim % 4 == 0 && prep->rope_dim <= a.c.head_dim,
                        "rope_dim must be a multiple of 4 up to head_dim");
                require(aligned(prep->d_rope, 16), "the rope table must be 16-byte aligned");
                require(prep->rope_len <= 0x7fffffffu, "rope_len is too large");
                a.rope = prep->d_rope;
                a.rope_dim = prep->rope_dim;
                a.rope_len = prep->rope_len;
                a.interleaved = prep->rope_interleaved ? 1 : 0;
            }
            require(aligned(prep->d_q_norm, 4) && aligned(prep->d_k_norm, 4), "norm weights must be 4-byte aligned");
            require(!(prep->d_q_norm || prep->d_k_norm) || (std::isfinite(prep->eps) && prep->eps >= 0.f),
                    "eps must be finite and not negative");
            a.q_norm = prep->d_q_norm;
            a.k_norm = prep->d_k_norm;
            a.eps = prep->eps;
        }
        if (!a.b.total || !a.b.n_seqs) return;
        check_pages(a.c);
        check_lists(a.b);
        const uint64_t width = (uint64_t)a.c.kv_heads * a.c.head_dim;
        check_rows(d_k, k_stride, width, es, "k");
        check_rows(d_v, v_stride, width, es, "v");
        require(aligned(d_err, 4), "d_err must be 4-byte aligned");
        if (d_q || d_q_out) {
            require(heads >= 1 && heads <= 65535, "heads must be 1..65535");
            check_rows(d_q, q_stride, (uint64_t)heads * a.c.head_dim, es, "q");
            check_rows(d_q_out, q_out_stride, (uint64_t)heads * a.c.head_dim, es, "q_out");
            require(d_q != d_q_out || q_stride == q_out_stride, "q made ready in place needs one stride");
            require(d_q == d_q_out || q_stride != q_out_stride ||
                        !share_memory(d_q, d_q_out, a.b.total, (uint64_t)heads * a.c.head_dim * es, q_stride * es),
                    "q_out may be q, but must not overlap it otherwise");
            a.heads = heads;
            a.q = d_q;
            a.q_out = d_q_out;
            a.q_stride = q_stride;
            a.q_out_stride = q_out_stride;
        }
        a.k = d_k;
        a.v = d_v;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.err = d_err;
        OnDeviceOf on(d_k);
        cuda_check(launch_kv8_append(a, sm_count(on.dev), static_cast<cudaStream_t>(stream)), "kv8 append");
    });
}

evl_status evl_kv8_attention_workspace_bytes(const evl_kv8_cache* cache, const evl_kv8_batch* batch, uint32_t type,
                                             uint32_t heads, size_t* bytes) {
    return guarded([&] {
        require(bytes, "null argument");
        elem_bytes(type);
        const Kv8Cache c = cache_of(cache);
        const Kv8Batch b = batch_of(batch);
        require(heads >= 1 && heads % c.kv_heads == 0, "heads must be a multiple of kv_heads");
        int dev = 0;
        cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
        *bytes = (size_t)kv8_attention_ws_bytes(c, b, heads, type, sm_count(dev));
    });
}

evl_status evl_kv8_attention(const evl_kv8_cache* cache, const evl_kv8_batch* batch, uint32_t type, const void* d_q,
                             uint64_t q_stride, uint32_t heads, float scale, void* d_out, uint64_t out_stride,
                             void* d_workspace, size_t workspace_bytes, int32_t* d_err, void* stream) {
    return guarded([&] {
        const uint64_t es = elem_bytes(type);
        Kv8AttnArgs a;
        a.c = cache_of(cache);
        a.b = batch_of(batch);
        require(heads >= 1 && heads <= 65535 && heads % a.c.kv_heads == 0, "heads must be a multiple of kv_heads");
        require(std::isfinite(scale), "scale must be finite");
        if (!a.b.total || !a.b.n_seqs) return;
        check_pages(a.c);
        check_lists(a.b);
        const uint64_t width = (uint64_t)heads * a.c.head_dim;
        check_rows(d_q, q_stride, width, es, "q");
        check_rows(d_out, out_stride, width, es, "out");
        require(aligned(d_err, 4), "d_err must be 4-byte aligned");
        OnDeviceOf on(d_q);
        const int sms = sm_count(on.dev);
        const uint64_t need = kv8_attention_ws_bytes(a.c, a.b, heads, type, sms);
        if (need) {
            require(d_workspace && aligned(d_workspace, 256), "workspace must be 256-byte aligned");
            require(workspace_bytes >= need, "workspace too small; size it with evl_kv8_attention_workspace_bytes");
        }
        a.type = type;
        a.heads = heads;
        a.q = d_q;
        a.out = d_out;
        a.q_stride = q_stride;
        a.out_stride = out_stride;
        a.scale = scale == 0.f ? 1.0f / std::sqrt((float)a.c.head_dim) : scale;
        a.ws = static_cast<uint8_t*>(d_workspace);
        a.err = d_err;
        cuda_check(launch_kv8_attention(a, sms, static_cast<cudaStream_t>(stream)), "kv8 attention");
    });
}

}  // extern "C"
