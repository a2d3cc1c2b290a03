// Operators of the decode path: norm and rotation of queries and keys (qk_norm_rope.cu), the 8-bit
// key/value cache (kv_cache.cu), attention over it (cache_attention.cu), 4-bit weights (q4.cu).
#pragma once
#include "launch.hpp"

namespace wgf {

// How a row of `dim` values is spread over lanes: the widest vector that all of `ptrs` (element addresses) and
// `strides` (in elements) allow, lanes per row and chunks per lane.
struct RowSpread {
    int vec, lanes, chunks;
};
RowSpread head_spread(DType dt, int64_t dim, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides);
constexpr int64_t kMaxNormDim = 512;

// Each head of q [.., seq, dim] and k (same rank 3 or 4, its own number of heads) normed, scaled by its weight and
// rotated by rows start, start + 1, ... of cos / sin.  One new buffer: q's result, then k's from element
// `k_offset` on, both dense.
TensorData run_qk_norm_rope(Device& dev, const TensorData& q, const TensorData& k, const TensorData& wq, const TensorData& wk,
                            const TensorData& cos, const TensorData& sin, float eps, int64_t start, int64_t k_offset);
// Where k's result starts in that buffer: behind q's, at a multiple of 8 elements.
inline int64_t qk_second_offset(int64_t q_numel) { return (q_numel + 7) / 8 * 8; }

// ---- 8-bit key/value cache ---------------------------------------------------------------------------------
// For every sequence, kv head and block of 64 tokens: the codes of the keys and of the values in the order in
// which the attention kernel's lanes read them (kv_cache.cu), and one scale each.  Beside them the
// tokens of the last two blocks in the element type, from which the open block's codes are made anew
// whenever tokens come to it: the codes never depend on how the tokens were appended.
struct KvCache : std::enable_shared_from_this<KvCache> {
    static constexpr int kBlock = 64;
    DeviceRef dev;
    DType dtype = DType::F32;
    int64_t batch = 0, heads = 0, dim = 0, dim_pad = 0, capacity = 0, blocks = 0;
    BufferRef codes;    // u8 [batch][heads][blocks][key, value][64 * dim_pad]
    BufferRef scales;   // f32 [batch][heads][blocks][key, value]
    BufferRef tail;     // dtype [batch][heads][block & 1][key, value][64][dim]
    BufferRef lens;     // i32 [batch] tokens, [batch] counts of the call
    // What the device's `lens` will hold once all queued work has run.
    std::vector<int64_t> lengths;
    // First block whose tokens are still held in the element type, per sequence.
    std::vector<int64_t> held_from;
    int64_t longest() const;
    // Tokens that the recording under way adds to every sequence (0 outside one).
    int64_t recorded_tokens() const;
};
using KvCacheRef = std::shared_ptr<KvCache>;

KvCacheRef kv_cache_create(const DeviceRef& dev, DType dtype, int64_t batch, int64_t heads, int64_t dim, int64_t capacity);
void kv_cache_truncate(KvCache& c, const int64_t* lengths);
// k, v [batch, heads, t, dim]; counts: how many of the t tokens each sequence gets, or null for all.
void kv_cache_append(KvCache& c, const TensorData& k, const TensorData& v, const int64_t* counts);
// The same behind norm and rotation of q and k at each sequence's own positions; returns q's result [batch, q_heads, t, dim].
TensorData kv_cache_append_qk(KvCache& c, const TensorData& q, const TensorData& k, const TensorData& v, const TensorData& wq,
                              const TensorData& wk, const TensorData& cos, const TensorData& sin, float eps, const int64_t* counts);
// The values that the codes stand for: [batch, heads, longest length, dim], zero behind each sequence's end.
void kv_cache_read(KvCache& c, TensorData& k, TensorData& v);
// softmax(scale q K^T) V for q [batch, q_heads, t, dim] at the last t positions of each sequence, each query
// seeing the keys up to its own position.
TensorData kv_cache_attention(KvCache& c, const TensorData& q, float scale, const int64_t* counts);
// Stores counts (or -1 for "all of the call's tokens") in the second half of c.lens.
void kv_cache_set_counts(KvCache& c, const int64_t* counts, int64_t t, const char* what);

// ---- 4-bit weights -----------------------------------------------------------------------------------------
// [n, k] as codes 0..15 in tiles of 16 rows and 64 columns, in the order in which the lanes of the product read them
// (q4.cu); value = scale * (code - 8), one scale for each row and `group` columns.
struct Q4Weight {
    DeviceRef dev;
    int64_t n = 0, k = 0, group = 0;
    int64_t row_tiles = 0, chunks = 0, groups = 0;   // tiles of 16 rows, of 64 columns, groups of a row
    DType scale_dtype = DType::F32;
    BufferRef codes;    // u32 [row_tiles][chunks][lane][4]
    BufferRef scales;   // scale_dtype [row_tiles][groups][16]
};
using Q4Ref = std::shared_ptr<Q4Weight>;

Q4Ref q4_quantize(const DeviceRef& dev, const TensorData& w, int64_t group);
Q4Ref q4_from_host(const DeviceRef& dev, int64_t n, int64_t k, int64_t group, const uint8_t* codes, DType scale_dtype, const void* scales);
TensorData q4_dequantize(Device& dev, const Q4Weight& w, DType dtype);
// x [.., k] times the transposed weights: [.., n]
TensorData run_matmul_q4(Device& dev, const TensorData& x, const Q4Weight& w);

}  // namespace wgf
