// int8.h -- host-side launchers and argument blocks of the 8-bit serving operators:
// quantised activation rows, the integer product with token and channel scales, and the
// 8-bit paged KV cache (append and attention).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace evl {

// A group of values whose largest magnitude is below this is stored as zeros (scale 0): the
// scale and its reciprocal then stay normal f32 numbers.
constexpr float kInt8Tiny = 7.888609052210118e-31f;  // 2^-100

// ---------------------------------------------------------------- int8_rows.cu
struct QuantRowsArgs {
    const void* x = nullptr;
    uint32_t type = 0;       // GGML_F32, GGML_F16 or GGML_BF16
    uint64_t x_stride = 0;   // elements between rows
    uint32_t rows = 0, cols = 0;
    int8_t* codes = nullptr;
    uint64_t code_stride = 0;  // bytes between rows
    float* scales = nullptr;
};
cudaError_t launch_quantize_rows(const QuantRowsArgs& a, int sms, cudaStream_t s);

// ---------------------------------------------------------------- int8_gemm.cu
struct I8GemmArgs {
    const int8_t* x = nullptr;  // [rows][x_stride]
    uint64_t x_stride = 0;
    const float* xs = nullptr;  // [rows]
    const int8_t* w = nullptr;  // [out][w_stride]
    uint64_t w_stride = 0;
    const float* ws = nullptr;  // [out]
    uint32_t rows = 0, out = 0, cols = 0;
    uint32_t type = 0;          // of y and add
    const void* add = nullptr;
    uint64_t add_stride = 0;    // elements
    void* y = nullptr;
    uint64_t y_stride = 0;      // elements
    int32_t* err = nullptr;     // optional
};
cudaError_t launch_i8_gemm(const I8GemmArgs& a, int sms, cudaStream_t s);
// How that launch cuts the product on the current device: tokens of a tile (0: CTA pairs, 256 x 256) and CTAs that share
// its K. By rows, out, cols, type and whether there is an addition.
void i8_gemm_cut(const I8GemmArgs& a, int sms, uint32_t& tokens, uint32_t& split);

// ---------------------------------------------------------------- kv8_append.cu, kv8_attention.cu
struct Kv8Cache {
    uint32_t kv_heads = 0, head_dim = 0, page_size = 0, n_pages = 0;
    int8_t *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;
    uint64_t page_stride = 0, scale_stride = 0;
};
struct Kv8Batch {
    uint32_t n_seqs = 0, total = 0, max_new = 0, max_len = 0, table_stride = 0;
    const int32_t *table = nullptr, *cu = nullptr, *len = nullptr;
};
struct Kv8AppendArgs {
    Kv8Cache c;
    Kv8Batch b;
    uint32_t type = 0, heads = 0;
    const void *k = nullptr, *v = nullptr, *q = nullptr;
    void* q_out = nullptr;
    uint64_t k_stride = 0, v_stride = 0, q_stride = 0, q_out_stride = 0;  // elements between tokens
    const float* rope = nullptr;  // [rope_len][rope_dim / 2][cos, sin]
    uint32_t rope_dim = 0, rope_len = 0, interleaved = 0;
    const float *q_norm = nullptr, *k_norm = nullptr;
    float eps = 0.f;
    int32_t* err = nullptr;
};
cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int sms, cudaStream_t s);

struct Kv8AttnArgs {
    Kv8Cache c;
    Kv8Batch b;
    uint32_t type = 0, heads = 0;
    const void* q = nullptr;
    void* out = nullptr;
    uint64_t q_stride = 0, out_stride = 0;  // elements between tokens
    float scale = 0.f;
    uint8_t* ws = nullptr;
    int32_t* err = nullptr;
};
uint64_t kv8_attention_ws_bytes(const Kv8Cache& c, const Kv8Batch& b, uint32_t heads, uint32_t type, int sms);
cudaError_t launch_kv8_attention(const Kv8AttnArgs& a, int sms, cudaStream_t s);

}  // namespace evl
