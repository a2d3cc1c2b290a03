// Norm of every head of the queries and keys, and the rotation by position, in one pass and one launch.
//
//   y = x / sqrt(mean_d(x^2) + eps) * w                      (each head by itself, w shared by the heads)
//   out[d] = y[d] cos - y[d + D/2] sin,  out[d + D/2] = y[d + D/2] cos + y[d] sin   for d < D/2
//
// All in f32, rounded once to the element type.  Every value is read once and written once: memory is the bound.
// A group of lanes holds a whole row (8 lanes for 128 values of 16 bits: two 16-byte loads each, the
// second being the rotation's partner of the first), so the mean needs three shuffles and no shared memory.
// A group takes HEADS heads of one token: their loads are all issued before the first is used, and the products of
// weights with cosines and sines are made once for them.
// 8 x 2048 tokens of 32 + 8 heads of 128, f16, 336 MB: 61.5 to 65.7 us by card (5.1 to 5.5 TB/s, 0.78 to 0.83 of the measured copy); with blocks of 256
// threads 70, with two heads a group 72 to 102, and 118 where rows were turned into f32 as they came (twice the registers).
#include <algorithm>

#include "decode.hpp"
#include "decode_common.cuh"

namespace wgf {

using namespace decode;

RowSpread head_spread(DType dt, int64_t dim, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
    const int64_t es = (int64_t)dtype_size(dt), half = dim / 2;
    for (int64_t v : {(int64_t)8, (int64_t)4, (int64_t)1}) {
        if (v * es > 16 || half % v) continue;
        bool ok = true;
        for (const void* p : ptrs) ok = ok && (uintptr_t)p % (uintptr_t)(v * es) == 0;
        for (int64_t s : strides) ok = ok && s % v == 0;
        if (!ok && v > 1) continue;
        const int64_t need = (half + v - 1) / v;
        int lanes = 1;
        while (lanes < 32 && lanes < need) lanes *= 2;
        return {(int)v, lanes, (int)((need + lanes - 1) / lanes)};
    }
    return {1, 32, 8};
}

namespace {

constexpr int kThreads = 64;     // short blocks: their loads, sums and stores lie at different times
constexpr int kHeads = 4;        // heads of a token that a group of lanes takes where there are enough tokens

struct QkParams {
    const void *x[2], *w[2], *cos, *sin;
    void* out[2];
    long long sb[2], sh[2], ss[2];   // strides of batch, head, token in elements
    long long cs_c, cs_s;            // row strides of cos / sin
    int heads[2], chunks0;           // heads of q and of k; groups of heads that belong to q
    int S, tokens, half, lanes;      // tokens = batch * S
    long long start;
    float eps;
};

template <typename T, int VEC, int NCH, int HEADS>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
    typedef HeadRow<T, VEC, NCH> Row;
    const int lane = threadIdx.x & (p.lanes - 1);
    const int per_block = kThreads / p.lanes;
    const int token = blockIdx.x * per_block + threadIdx.x / p.lanes;
    const int which = (int)blockIdx.y >= p.chunks0;
    const int h0 = ((int)blockIdx.y - (which ? p.chunks0 : 0)) * HEADS;
    const int heads = p.heads[which];
    const bool live = token < p.tokens;
    const int t = live ? token : 0;                       // idle groups run along for the shuffles
    const int b = t / p.S, s = t - b * p.S;
    const T* x = (const T*)p.x[which] + b * p.sb[which] + s * p.ss[which];
    Row r[HEADS];
    x += (long long)h0 * p.sh[which];
#pragma unroll
    for (int u = 0; u < HEADS; ++u) r[u].load(x + (long long)min(u, heads - 1 - h0) * p.sh[which], p.half, lane, p.lanes);
    Turn<T, VEC, NCH> turn;
    turn.load((const T*)p.w[which], (const T*)p.cos + (p.start + s) * p.cs_c, (const T*)p.sin + (p.start + s) * p.cs_s, p.half, lane, p.lanes);
    const long long step = (long long)p.S * (2ll * p.half);
    T* out = (T*)p.out[which] + ((long long)b * heads * p.S + s) * (2ll * p.half) + h0 * step;
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
        const Row y = r[u].turned(turn, r[u].inverse_rms(p.half, p.lanes, p.eps));
        if (live && h0 + u < heads) y.store(out + u * step, p.half, lane, p.lanes);
    }
}

template <typename T, int VEC, int NCH>
void launch_qk(Device& dev, QkParams& p) {
    const int per_block = kThreads / p.lanes;
    const unsigned bx = (unsigned)((p.tokens + per_block - 1) / per_block);
    const bool many = NCH <= 2 && (long long)bx * ((p.heads[0] + kHeads - 1) / kHeads + (p.heads[1] + kHeads - 1) / kHeads) >= 8ll * dev.sm_count;
    const int u = many ? kHeads : 1;
    p.chunks0 = (p.heads[0] + u - 1) / u;
    const dim3 grid(bx, (unsigned)(p.chunks0 + (p.heads[1] + u - 1) / u));
    dev.begin_launch("qk_norm_rope");
    if (!dev.dry) {
        if constexpr (NCH <= 2) {
            if (many) qk_norm_rope_kernel<T, VEC, NCH, kHeads><<<grid, kThreads, 0, dev.stream>>>(p);
        }
        if (!many) qk_norm_rope_kernel<T, VEC, NCH, 1><<<grid, kThreads, 0, dev.stream>>>(p);
    }
    dev.end_launch();
}

template <typename T>
void dispatch_qk(Device& dev, QkParams& p, const RowSpread& s) {
    constexpr int W = 16 / (int)sizeof(T);   // widest vector
    if (s.vec == W && s.chunks == 1) launch_qk<T, W, 1>(dev, p);
    else if (s.vec == W && s.chunks == 2) launch_qk<T, W, 2>(dev, p);
    else if (s.vec == 4 && s.chunks <= 2) launch_qk<T, 4, 2>(dev, p);
    else launch_qk<T, 1, 8>(dev, p);
}

}  // namespace

TensorData run_qk_norm_rope(Device& dev, const TensorData& q_in, const TensorData& k_in, const TensorData& wq_in, const TensorData& wk_in,
                            const TensorData& cos_in, const TensorData& sin_in, float eps, int64_t start, int64_t k_offset) {
    dev.make_current();
    const int r = q_in.layout.rank();
    const int64_t S = q_in.layout.shape[r - 2], D = q_in.layout.shape[r - 1];
    auto last_dense = [&](const TensorData& t) {
        const int l = t.layout.rank() - 1;
        return t.layout.strides[l] == 1 || t.layout.shape[l] == 1 ? t : run_compact(dev, t);
    };
    const TensorData x[2] = {last_dense(q_in), last_dense(k_in)}, w[2] = {last_dense(wq_in), last_dense(wk_in)};
    const TensorData cos = last_dense(cos_in), sin = last_dense(sin_in);
    for (const TensorData* t : {&x[0], &x[1], &w[0], &w[1], &cos, &sin}) dev.wait_for(*t->buf);
    const int64_t nq = q_in.layout.numel(), nk = k_in.layout.numel();
    TensorData out;
    out.dtype = q_in.dtype;
    out.layout = Layout::contiguous({k_offset + nk});
    out.buf = dev.alloc((size_t)std::max<int64_t>(k_offset + nk, 1) * dtype_size(out.dtype), false);
    if (nq + nk == 0) return out;
    QkParams p{};
    const int64_t B = r == 4 ? q_in.layout.shape[0] : 1;
    WGF_CHECK(B * S < (1ll << 30) && q_in.layout.shape[r - 3] + k_in.layout.shape[r - 3] <= 65535, WGF_ERR_UNSUPPORTED, "qk_norm_rope: 2^30 tokens or more, or more than 65535 heads");
    for (int i = 0; i < 2; ++i) {
        p.x[i] = x[i].base_ptr();
        p.w[i] = w[i].base_ptr();
        p.out[i] = (char*)out.buf->ptr + (i ? k_offset : 0) * (int64_t)dtype_size(out.dtype);
        p.sb[i] = r == 4 ? x[i].layout.strides[0] : 0;
        p.sh[i] = x[i].layout.strides[r - 3];
        p.ss[i] = x[i].layout.strides[r - 2];
        p.heads[i] = (int)x[i].layout.shape[r - 3];
    }
    p.cos = cos.base_ptr();
    p.sin = sin.base_ptr();
    p.cs_c = cos.layout.strides[0];
    p.cs_s = sin.layout.strides[0];
    p.S = (int)S;
    p.tokens = (int)(B * S);
    p.half = (int)(D / 2);
    p.start = start;
    p.eps = eps;
    const RowSpread s = head_spread(out.dtype, D, {p.x[0], p.x[1], p.w[0], p.w[1], p.cos, p.sin, p.out[0], p.out[1]},
                                    {p.sb[0], p.sb[1], p.sh[0], p.sh[1], p.ss[0], p.ss[1], p.cs_c, p.cs_s});
    p.lanes = s.lanes;
    if (out.dtype == DType::F32) dispatch_qk<float>(dev, p, s);
    else if (out.dtype == DType::F16) dispatch_qk<__half>(dev, p, s);
    else dispatch_qk<__nv_bfloat16>(dev, p, s);
    return out;
}

}  // namespace wgf
