// 8-bit key/value cache: filling it, rolling it back and reading it.
//
// A block is 64 tokens of one sequence and kv head.  Its keys, and by themselves its values, share a scale:
//   scale = max|x| / 127,   code = round(127 x / max|x|)  (ties to even, as if the quotient were exact),
// with max|x| taken as at least 2^-100, and a NaN scale (codes 0) where a value is not finite.  A code stands for
// code * scale.  The open block, the one that the next token goes to, is coded anew from its tokens' own values
// with every append; those are kept for two blocks ("tail"), so that the last 64 tokens at least can be taken
// back.  The state is therefore a function of the tokens alone, and no value is rounded twice.
//
// Codes are stored as code + 128 in the order in which cache_attention.cu's lanes read them, 16 bytes a lane:
//   keys    [token group nt 0..7][dims / 64][lane][16]: lane (g, c) has 16 dims, c * 16 on, of token
//           16 (g / 2) + 4 (nt / 2) + 2 (nt % 2) + g % 2
//   values  [dims / 8][lane][16]: lane (g, c) has tokens 16 c .. 16 c + 15 of dim 8 nd + g
// Dims are padded to a multiple of 64 by zeros.
//
// The append kernel: one CTA for each (sequence, head, block touched, keys or values).  It gathers the block's tokens
// in shared memory (old ones from the tail, new ones from the call, keys behind norm and rotation if asked), finds the
// largest magnitude on the way and writes the codes; for long prompts it is bound by memory, for one token by
// the latency of one load, one reduction and one store.
// 4 sequences of up to 2048 tokens, 8 heads of 128, bf16, 79 MB in and out: an append into an emptied cache and a read of it take 36 to 37 us,
// 20 in the append kernel and 13 in the read, both bound by the instructions that turn values into codes and into the lanes' order
// (about 30 a value) and back, not by memory, which would need 12 for both.
#include <algorithm>

#include "decode.hpp"
#include "decode_common.cuh"

namespace wgf {

using namespace decode;

namespace {

constexpr int kBlock = KvCache::kBlock;
constexpr int kThreads = 256;
constexpr int kGiven = 256;
constexpr int kRecode = 1 << 30;

struct CacheView {
    uint8_t* codes;
    float* scales;
    void* tail;
    int* lens;                 // [batch] lengths, [batch] counts
    int batch, heads, dim, dim_pad, blocks, capacity;
    __device__ uint8_t* block(int b, int h, int blk, int kv) const {
        return codes + ((((long long)b * heads + h) * blocks + blk) * 2 + kv) * (long long)(kBlock * dim_pad);
    }
    __device__ float* scale(int b, int h, int blk, int kv) const {
        return scales + (((long long)b * heads + h) * blocks + blk) * 2 + kv;
    }
    template <typename T> __device__ T* tail_of(int b, int h, int blk, int kv) const {
        return (T*)tail + (((((long long)b * heads + h) * 2 + (blk & 1)) * 2 + kv) * kBlock) * (long long)dim;
    }
};

struct AppendParams {
    CacheView c;
    const void *k, *v;                     // [batch, heads, t, dim]
    long long kb, kh, ks, vb, vh, vs;      // strides of batch, head, token
    int t;                                 // new tokens a sequence; -1: none, sequences with a count are coded anew
    int use_counts;                        // 1: in the second half of the cache's lens, 2: in `given`
    int blocks_touched;                    // of one sequence, at most
    // keys behind norm and rotation, and the queries with them
    const void *wk, *wq, *cos, *sin, *q;
    void* q_out;
    long long qb, qh, qs, cs_c, cs_s;
    int q_heads, q_lanes, lanes, table_rows;
    unsigned kv_ctas;                      // CTAs behind these do rows of q
    float eps;
    unsigned* ticket;
    // Small batches' numbers by value, so that they cost no launch of their own: counts, or (t < 0) the new lengths, with
    // kRecode where the open block's codes have to be made anew.
    int given[kGiven];
};

__device__ __forceinline__ int key_token(int nt, int g) { return (g >> 1) * 16 + (nt >> 1) * 4 + (nt & 1) * 2 + (g & 1); }

// The block's tokens in shared memory: rows of dim_pad values in 16-byte pieces, the pieces of a row exchanged so that the
// lanes of neither reading below, of eight tokens' pieces or of four groups of 16 tokens, meet in a bank.
template <typename T, int DP> __device__ __forceinline__ int tile_at(int row, int j) {
    constexpr int PIECE = 16 / (int)sizeof(T);
    const int turn = sizeof(T) == 2 ? ((row >> 4) & 3) * 2 | (row & 1) : ((row >> 4) & 1) * 4 | (row & 1);
    return row * DP + (j ^ (turn * PIECE));
}

// The largest |x|: two 16-bit ones side by side, or the bits of an f32.  As an ordered integer NaN is above infinity is above
// every number; the maximum of pairs keeps a NaN.
template <typename T> struct Largest {
    unsigned top = 0;
    template <int VEC> __device__ __forceinline__ void take(const Pack<T, VEC>& x) {
        if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
            typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
            const T2* w = reinterpret_cast<const T2*>(&x);
            T2 t = *reinterpret_cast<const T2*>(&top);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) t = __hmax2_nan(t, __habs2(w[i]));
            top = *reinterpret_cast<const unsigned*>(&t);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if constexpr (sizeof(T) == 2) top = max(top, *reinterpret_cast<const unsigned short*>(&x.v[e]) & 0x7fffu);
                else top = max(top, abs_bits(x.v[e]));
            }
        }
    }
    // as the bits of an f32
    __device__ __forceinline__ unsigned bits() const {
        if constexpr (sizeof(T) == 2) {
            const unsigned short h = (unsigned short)max(top & 0xffffu, top >> 16);
            return abs_bits(to_f<T>(*reinterpret_cast<const T*>(&h)));
        } else {
            return top;
        }
    }
};

// Gathers block `blk` into the tile (zero where it has no token) and returns this thread's largest |x| as the bits of an f32.
// Tokens before `len` come from the tail, those up to `end` from the call.  With `keep`, new tokens go to the tail as well.
template <typename T, int DP, int VEC, int NCH, bool NORM>
__device__ unsigned gather(const AppendParams& p, T* tile, int b, int h, int blk, int kv, int len, int end, bool keep) {
    const CacheView& c = p.c;
    Largest<T> top;
    const int first = blk * kBlock;
    const T* src = kv ? (const T*)p.v + b * p.vb + h * p.vh : (const T*)p.k + b * p.kb + h * p.kh;
    const long long step = kv ? p.vs : p.ks;
    T* tail = c.tail_of<T>(b, h, blk, kv);
    typedef Pack<T, VEC> V;
    const bool turned = NORM && kv == 0;
    // a thread's pieces, one row and column behind the other; four loads at a time
    constexpr int per_row = DP / VEC, row_step = kThreads / per_row, j_step = (kThreads - row_step * per_row) * VEC;
    int row = threadIdx.x / per_row, j = (threadIdx.x - row * per_row) * VEC;
    while (row < kBlock) {
        V x[4];
        int rows[4], js[4];
        bool mine[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            rows[i] = row;
            js[i] = j;
            const int pos = first + row;
            mine[i] = row < kBlock && !(turned && j < c.dim && pos >= len && pos < end);      // those are written below
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[i].v[e] = from_f<T>(0.f);
            if (mine[i] && j < c.dim && pos < end)
                x[i] = *reinterpret_cast<const V*>(pos < len ? tail + (long long)row * c.dim + j : src + (long long)(pos - len) * step + j);
            row += row_step;
            j += j_step;
            if (j_step && j >= DP) {
                j -= DP;
                ++row;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!mine[i]) continue;
            top.take(x[i]);
            *reinterpret_cast<V*>(tile + tile_at<T, DP>(rows[i], js[i])) = x[i];
            const int pos = first + rows[i];
            if (keep && js[i] < c.dim && pos >= len && pos < end) *reinterpret_cast<V*>(tail + (long long)rows[i] * c.dim + js[i]) = x[i];
        }
    }
    if (turned) {
        typedef HeadRow<T, VEC, NCH> Row;
        const int half = c.dim / 2, lane = threadIdx.x & (p.lanes - 1), groups = kThreads / p.lanes;
        const int begin = max(len, first), stop = min(end, first + kBlock);
        for (int base = begin; base < stop; base += groups) {      // all lanes of a warp stay together for the shuffles
            const int pos = base + threadIdx.x / p.lanes;
            const bool live = pos < stop;
            const int at = live ? pos : begin;
            Row r;
            r.load(src + (long long)(at - len) * step, half, lane, p.lanes);
            Turn<T, VEC, NCH> turn;
            const long long angle = min(at, p.table_rows - 1);
            turn.load((const T*)p.wk, (const T*)p.cos + angle * p.cs_c, (const T*)p.sin + angle * p.cs_s, half, lane, p.lanes);
            r = r.turned(turn, r.inverse_rms(half, p.lanes, p.eps));
            if (!live) continue;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
                const int j = (lane + n * p.lanes) * VEC;
                if (j >= half) continue;
                // the values that the operators one by one would hand over: rounded to the type
                top.take(r.lo[n]);
                top.take(r.hi[n]);
                *reinterpret_cast<V*>(tile + tile_at<T, DP>(pos - first, j)) = r.lo[n];
                *reinterpret_cast<V*>(tile + tile_at<T, DP>(pos - first, half + j)) = r.hi[n];
            }
            if (keep) r.store(tail + (long long)(pos - first) * c.dim, half, lane, p.lanes);
        }
    }
    return top.bits();
}

__device__ __noinline__ unsigned four_exact(float x0, float x1, float x2, float x3, float num, float den, float inv) {
    return (unsigned)(exact_code(x0, num, den, inv) + 128) | (unsigned)(exact_code(x1, num, den, inv) + 128) << 8 |
           (unsigned)(exact_code(x2, num, den, inv) + 128) << 16 | (unsigned)(exact_code(x3, num, den, inv) + 128) << 24;
}
// Four values' codes + 128 as bytes.  x k is off by less than 2^-16, so the nearest whole number is the code unless the product is
// that near to a border; `border` then tells, and the four are done over with exact_code.  Adding 1.5 * 2^23 + 128 leaves the
// whole number in the low bits.
struct Coder {
    float k;            // 127 / max|x|
    float num, den, inv;
    static __device__ __forceinline__ float magic() { return 12582912.f + 128.f; }
    __device__ __forceinline__ unsigned four(const float (&x)[4]) const {
        float m[4], off = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = __fmaf_rn(x[i], k, magic());
            off = fmaxf(off, fabsf(__fmaf_rn(x[i], k, -(m[i] - magic()))));
        }
        if (off > 0.5f - 0x1p-15f) return four_exact(x[0], x[1], x[2], x[3], num, den, inv);
        const unsigned a = __byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040), b = __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040);
        return __byte_perm(a, b, 0x5410);
    }
};

template <typename T, int DP, int VEC, int NCH, bool NORM>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ AppendParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ unsigned warp_top[kThreads / 32];
    __shared__ unsigned last;
    const CacheView& c = p.c;
    if (blockIdx.x < p.kv_ctas) {
        unsigned i = blockIdx.x;
        const int kv = i & 1;
        i >>= 1;
        const int nb = i % p.blocks_touched;
        i /= p.blocks_touched;
        const int h = i % c.heads, b = i / c.heads;
        const int len = p.t < 0 && p.use_counts == 2 ? p.given[b] & (kRecode - 1) : c.lens[b];
        const int asked = p.use_counts == 2 ? (p.t < 0 ? p.given[b] >> 30 : p.given[b]) : p.use_counts ? c.lens[c.batch + b] : p.t;
        if (p.t < 0 && p.use_counts == 2 && nb + h + kv == 0 && threadIdx.x == 0) c.lens[b] = len;
        const int fresh = p.t < 0 ? 0 : min(asked, c.capacity - len);
        const int end = len + fresh, blk = len / kBlock + nb;
        T* tile = (T*)smem;
        if (p.t < 0 ? (asked > 0 && nb == 0 && len % kBlock != 0) : (fresh > 0 && blk * kBlock < end)) {
            // the two blocks that the tail keeps: the open one and the one before it
            const int open = end / kBlock, first_blk = len / kBlock;
            // a block of the same parity as the first one would overwrite what the first one's CTA reads: that CTA
            // writes it, after it has read
            const bool keep = blk >= open - 1 && (blk == first_blk || ((blk ^ first_blk) & 1));
            unsigned top = gather<T, DP, VEC, NCH, NORM>(p, tile, b, h, blk, kv, len, end, keep && p.t > 0);
            top = __reduce_max_sync(0xffffffffu, top);
            if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
            __syncthreads();
            top = warp_top[0];
#pragma unroll
            for (int w = 1; w < kThreads / 32; ++w) top = max(top, warp_top[w]);
            const bool finite = top < 0x7f800000u;
            const float amax = fmaxf(__uint_as_float(finite ? top : 0u), 0x1p-100f);
            // far up, 127 x would leave the range: both sides of the quotient come down by the same power of two
            const float down = amax > 0x1p100f ? 0x1p-32f : 1.f;
            Coder code;
            code.k = finite ? 127.f / amax : 0.f;
            code.num = finite ? 127.f * down : 0.f;
            code.den = amax * down;
            code.inv = 1.f / code.den;
            uint4* out = reinterpret_cast<uint4*>(c.block(b, h, blk, kv));
            const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            if (kv == 0) {
                // 16 dims of a token
                for (int i = threadIdx.x; i < kBlock * (DP / 16); i += kThreads) {
                    const int lane = i & 31, j = (i >> 5) % (DP / 64), nt = (i >> 5) / (DP / 64);
                    const int row = key_token(nt, lane >> 2), at = j * 64 + (lane & 3) * 16;
                    unsigned w[4];
#pragma unroll
                    for (int q = 0; q < 16; q += 16 / (int)sizeof(T)) {
                        const Pack<T, 16 / sizeof(T)> x = *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(tile + tile_at<T, DP>(row, at + q));
#pragma unroll
                        for (int e = 0; e < 16 / (int)sizeof(T); e += 4) {
                            const float v[4] = {to_f<T>(x.v[e]), to_f<T>(x.v[e + 1]), to_f<T>(x.v[e + 2]), to_f<T>(x.v[e + 3])};
                            w[(q + e) / 4] = code.four(v);
                        }
                    }
                    out[i] = finite ? make_uint4(w[0], w[1], w[2], w[3]) : none;
                }
            } else {
                // 16 tokens of two dims side by side
                for (int i = threadIdx.x; i < kBlock * (DP / 32); i += kThreads) {
                    const int c4 = i & 3, d = (i >> 2) * 2;
                    unsigned w[2][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float v[2][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const Pack<T, 2> x = *reinterpret_cast<const Pack<T, 2>*>(tile + tile_at<T, DP>(c4 * 16 + q * 4 + e, d));
                            v[0][e] = to_f<T>(x.v[0]);
                            v[1][e] = to_f<T>(x.v[1]);
                        }
                        w[0][q] = code.four(v[0]);
                        w[1][q] = code.four(v[1]);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        out[(d >> 3) * 32 + ((d & 7) + e) * 4 + c4] = finite ? make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]) : none;
                }
            }
            // 127 times the quotient of the largest f32 would round to infinity: that one scale is the number below
            if (threadIdx.x == 0) *c.scale(b, h, blk, kv) = finite ? fminf(amax / 127.f, 0x1.020406p+121f) : __uint_as_float(0x7fc00000u);
            if (blk == first_blk && p.t > 0) {
                for (int x = max(open - 1, first_blk + 1); x <= open; ++x)
                    if (!((x ^ first_blk) & 1) && x * kBlock < end) {
                        __syncthreads();
                        gather<T, DP, VEC, NCH, NORM>(p, tile, b, h, x, kv, len, end, true);
                    }
            }
        }
    } else if constexpr (NORM) {
        typedef HeadRow<T, VEC, NCH> Row;
        const int half = c.dim / 2, lane = threadIdx.x & (p.q_lanes - 1), groups = kThreads / p.q_lanes;
        const long long rows = (long long)c.batch * p.q_heads * p.t;
        const long long row = (long long)(blockIdx.x - p.kv_ctas) * groups + threadIdx.x / p.q_lanes;
        const long long at = min(row, rows - 1);
        const int s = (int)(at % p.t);
        const long long o = at / p.t;
        const int h = (int)(o % p.q_heads), b = (int)(o / p.q_heads);
        const int len = c.lens[b], asked = p.use_counts == 2 ? p.given[b] : p.use_counts ? c.lens[c.batch + b] : p.t;
        Row r;
        r.load((const T*)p.q + b * p.qb + h * p.qh + s * p.qs, half, lane, p.q_lanes);
        Turn<T, VEC, NCH> turn;
        const long long angle = min(len + s, p.table_rows - 1);
        turn.load((const T*)p.wq, (const T*)p.cos + angle * p.cs_c, (const T*)p.sin + angle * p.cs_s, half, lane, p.q_lanes);
        r = r.turned(turn, r.inverse_rms(half, p.q_lanes, p.eps));
        if (row < rows) {
            if (s >= asked) {      // a padding row: zeros, whatever it held
#pragma unroll
                for (int n = 0; n < NCH; ++n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) r.lo[n].v[e] = r.hi[n].v[e] = from_f<T>(0.f);
            }
            r.store((T*)p.q_out + row * c.dim, half, lane, p.q_lanes);
        }
    }
    if (p.t < 0) return;
    // Everyone has read the lengths: the last CTA to get here moves them on.
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (last) {
        for (int b = threadIdx.x; b < c.batch; b += kThreads) {
            const int len = c.lens[b], asked = p.use_counts == 2 ? p.given[b] : p.use_counts ? c.lens[c.batch + b] : p.t;
            c.lens[b] = len + min(asked, c.capacity - len);
        }
        if (threadIdx.x == 0) *p.ticket = 0;
    }
}

// Numbers by value: nothing has to outlive the launch on the host, and a recording holds them as they are.
struct SetParams {
    int* to;
    int n;
    int v[896];
};
__global__ void kv_set_kernel(const __grid_constant__ SetParams p) {
    for (int i = threadIdx.x; i < p.n; i += blockDim.x) p.to[i] = p.v[i];
}

// The number that a byte stands for: it is put under the exponent of 2^23, and 2^23 + 128 is taken off
__device__ __forceinline__ float byte_code(unsigned w, int i) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | i)) - 8388736.f; }

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ CacheView c, T* __restrict__ k_out,
                                                           T* __restrict__ v_out, int longest, int out_blocks) {
    const int kv = blockIdx.x & 1;
    unsigned i = blockIdx.x >> 1;
    const int blk = i % out_blocks;
    i /= out_blocks;
    const int h = i % c.heads, b = i / c.heads;
    const int rows = min(kBlock, longest - blk * kBlock), have = min(max(c.lens[b] - blk * kBlock, 0), rows);
    T* out = (kv ? v_out : k_out) + (((long long)b * c.heads + h) * longest + blk * kBlock) * (long long)c.dim;
    const float scale = have > 0 ? *c.scale(b, h, blk, kv) : 0.f;
    const uint4* in = reinterpret_cast<const uint4*>(c.block(b, h, blk, kv));
    if (kv == 0) {
        // 16 dims of a token are 16 values in a row
        for (int n = threadIdx.x; n < kBlock * (DP / 16); n += kThreads) {
            const int lane = n & 31, j = (n >> 5) % (DP / 64), nt = (n >> 5) / (DP / 64);
            const int row = key_token(nt, lane >> 2), d = j * 64 + (lane & 3) * 16;
            if (row >= rows || d >= c.dim) continue;
            const uint4 u = row < have ? in[n] : make_uint4(0, 0, 0, 0);
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
            constexpr int W = 16 / (int)sizeof(T) < 8 ? 16 / (int)sizeof(T) : 8;
#pragma unroll
            for (int q = 0; q < 16; q += W) {
                if (d + q >= c.dim) break;                     // head_dim is a multiple of 8
                Pack<T, W> x;
#pragma unroll
                for (int e = 0; e < W; ++e) x.v[e] = from_f<T>(row < have ? byte_code(w[(q + e) >> 2], (q + e) & 3) * scale : 0.f);
                *reinterpret_cast<Pack<T, W>*>(out + (long long)row * c.dim + d + q) = x;
            }
        }
    } else {
        // 16 tokens of four dims: their bytes are turned four by four
        for (int n = threadIdx.x; n < DP; n += kThreads) {
            const int c4 = n / (DP / 4), d = n % (DP / 4) * 4;
            if (d >= c.dim || c4 * 16 >= rows) continue;
            uint4 u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = c4 * 16 < have ? in[(d >> 3) * 32 + ((d & 7) + e) * 4 + c4] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                unsigned w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = q == 0 ? u[e].x : q == 1 ? u[e].y : q == 2 ? u[e].z : u[e].w;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int row = c4 * 16 + q * 4 + t;
                    if (row >= rows) break;
                    Pack<T, 4> x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x.v[e] = from_f<T>(row < have ? byte_code(w[e], t) * scale : 0.f);
                    *reinterpret_cast<Pack<T, 4>*>(out + (long long)row * c.dim + d) = x;
                }
            }
        }
    }
}

CacheView view_of(const KvCache& c) {
    CacheView v{};
    v.codes = (uint8_t*)c.codes->ptr;
    v.scales = (float*)c.scales->ptr;
    v.tail = c.tail->ptr;
    v.lens = (int*)c.lens->ptr;
    v.batch = (int)c.batch;
    v.heads = (int)c.heads;
    v.dim = (int)c.dim;
    v.dim_pad = (int)c.dim_pad;
    v.blocks = (int)c.blocks;
    v.capacity = (int)c.capacity;
    return v;
}

// What a recording that appends does to the cache each time it is launched.
struct CacheStep : ReplayStep {
    KvCacheRef cache;
    int64_t added = 0;
    int64_t table_rows = INT64_MAX;   // rows of the position tables that the recording reads
    void check() const override {
        const int64_t n = cache->longest() + added;
        WGF_CHECK(n <= cache->capacity, WGF_ERR_INVALID_ARGUMENT,
                  "the recorded append does not fit: " + std::to_string(n) + " tokens in a cache for " + std::to_string(cache->capacity));
        WGF_CHECK(n <= table_rows, WGF_ERR_SHAPE, "the recorded append is past the end of its cos / sin tables");
    }
    void commit() override {
        for (size_t b = 0; b < cache->lengths.size(); ++b) {
            cache->lengths[b] += added;
            cache->held_from[b] = std::max(cache->held_from[b], cache->lengths[b] / kBlock - 1);
        }
    }
};

CacheStep* recorded_step(const KvCache& c) {
    for (auto& s : c.dev->recorded_steps())
        if (auto* mine = dynamic_cast<CacheStep*>(s.get()))
            if (mine->cache.get() == &c) return mine;
    return nullptr;
}

void note(KvCache& c) {
    for (const BufferRef& b : {c.codes, c.scales, c.tail, c.lens}) c.dev->note_recorded_buffer(b);
}

void set_ints(Device& dev, int* to, const std::vector<int>& v, const char* what) {
    for (size_t at = 0; at < v.size(); at += 896) {
        SetParams p{};
        p.to = to + at;
        p.n = (int)std::min<size_t>(896, v.size() - at);
        std::copy(v.begin() + at, v.begin() + at + p.n, p.v);
        dev.begin_launch(what);
        if (!dev.dry) kv_set_kernel<<<1, 256, 0, dev.stream>>>(p);
        dev.end_launch();
    }
}

template <typename F> void allow_smem(Device& dev, F kernel, size_t bytes) {
    // 48 KiB need no leave, what the kernels declare among them
    if (bytes > 47 * 1024 && !dev.dry) WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
}

template <typename F> void for_pad(int64_t dim_pad, F&& f) {
    switch (dim_pad) {
        case 64: return f(std::integral_constant<int, 64>());
        case 128: return f(std::integral_constant<int, 128>());
        case 192: return f(std::integral_constant<int, 192>());
        default: return f(std::integral_constant<int, 256>());
    }
}

template <typename T, int VEC, int NCH>
void launch_append(Device& dev, const AppendParams& p, unsigned q_ctas, bool norm, const char* what) {
    for_pad(p.c.dim_pad, [&](auto pad) {
        constexpr int DP = decltype(pad)::value;
        const size_t smem = (size_t)kBlock * DP * sizeof(T);
        auto go = [&](auto kernel) {
            allow_smem(dev, kernel, smem);
            dev.begin_launch(what);
            if (!dev.dry) kernel<<<p.kv_ctas + q_ctas, kThreads, smem, dev.stream>>>(p);
            dev.end_launch();
        };
        if (norm) go(kv_append_kernel<T, DP, VEC, NCH, true>);
        else go(kv_append_kernel<T, DP, VEC, NCH, false>);
    });
}

template <typename T>
void dispatch_append(Device& dev, const AppendParams& p, const RowSpread& s, unsigned q_ctas, bool norm, const char* what) {
    constexpr int W = 16 / (int)sizeof(T);
    if (s.vec == W) launch_append<T, W, 1>(dev, p, q_ctas, norm, what);        // dim <= 256: one chunk a lane
    else launch_append<T, 1, 4>(dev, p, q_ctas, norm, what);
}

void run_append(Device& dev, KvCache& c, AppendParams& p, const RowSpread& s, unsigned q_ctas, bool norm, const char* what) {
    const long long ctas = 2ll * c.batch * c.heads * p.blocks_touched;
    WGF_CHECK(ctas + q_ctas < (1ll << 31), WGF_ERR_UNSUPPORTED, "append of more than 2^30 blocks in one call");
    p.kv_ctas = (unsigned)ctas;
    p.ticket = (unsigned*)dev.counters();
    p.lanes = p.q_lanes = s.lanes;
    if (c.dtype == DType::F32) dispatch_append<float>(dev, p, s, q_ctas, norm, what);
    else if (c.dtype == DType::F16) dispatch_append<__half>(dev, p, s, q_ctas, norm, what);
    else dispatch_append<__nv_bfloat16>(dev, p, s, q_ctas, norm, what);
}

void check_new(const KvCache& c, const TensorData& x, const char* what) {
    WGF_CHECK(x.layout.rank() == 4, WGF_ERR_RANK, std::string(what) + " must be [batch, heads, tokens, head_dim]");
    WGF_CHECK(x.dtype == c.dtype, WGF_ERR_DTYPE, std::string(what) + " differs from the cache in element type");
}

// The two forms of append; q is null without norm and rotation.
TensorData append(KvCache& c, const TensorData& k_in, const TensorData& v_in, const int64_t* counts, const TensorData* q_in,
                  const TensorData* wq_in, const TensorData* wk_in, const TensorData* cos_in, const TensorData* sin_in, float eps) {
    Device& dev = *c.dev;
    check_new(c, k_in, "keys");
    check_new(c, v_in, "values");
    const int64_t t = k_in.layout.shape[2];
    WGF_CHECK(t < (1ll << 30), WGF_ERR_UNSUPPORTED, "append of 2^30 tokens or more");
    const std::vector<int64_t> want = {c.batch, c.heads, t, c.dim};
    WGF_CHECK(k_in.layout.shape == want && v_in.layout.shape == want, WGF_ERR_SHAPE,
              "keys and values must be [" + std::to_string(c.batch) + ", " + std::to_string(c.heads) + ", tokens, " + std::to_string(c.dim) + "]");
    int64_t most = 0;
    if (counts) {
        if (dev.recording()) fail(WGF_ERR_UNSUPPORTED, "counts of an append are fixed numbers: a recording takes none");
        for (int64_t b = 0; b < c.batch; ++b) {
            WGF_CHECK(counts[b] >= 0 && counts[b] <= t, WGF_ERR_INVALID_ARGUMENT, "a count is not between 0 and the number of tokens given");
            most = std::max(most, c.lengths[b] + counts[b]);
        }
    } else {
        most = c.longest() + c.recorded_tokens() + t;
    }
    WGF_CHECK(most <= c.capacity, WGF_ERR_INVALID_ARGUMENT,
              "append does not fit: " + std::to_string(most) + " tokens in a cache for " + std::to_string(c.capacity));
    TensorData out;
    if (q_in) {
        check_new(c, *q_in, "queries");
        const auto& qs = q_in->layout.shape;
        WGF_CHECK(qs[0] == c.batch && qs[2] == t && qs[3] == c.dim, WGF_ERR_SHAPE, "queries must be [batch, query heads, tokens, head_dim] like the keys");
        WGF_CHECK(c.dim % 2 == 0, WGF_ERR_UNSUPPORTED, "rotation needs an even head_dim");
        for (const TensorData* w : {wq_in, wk_in}) {
            WGF_CHECK(w->layout.rank() == 1 && w->layout.shape[0] == c.dim, WGF_ERR_SHAPE, "a head norm's weight must be [head_dim]");
            WGF_CHECK(w->dtype == c.dtype, WGF_ERR_DTYPE, "a head norm's weight differs in element type");
        }
        for (const TensorData* w : {cos_in, sin_in}) {
            WGF_CHECK(w->layout.rank() == 2 && w->layout.shape[1] * 2 == c.dim && w->layout.shape[0] == cos_in->layout.shape[0], WGF_ERR_SHAPE,
                      "cos / sin must be equal [positions, head_dim / 2]");
            WGF_CHECK(w->dtype == c.dtype, WGF_ERR_DTYPE, "cos / sin differ in element type");
        }
        WGF_CHECK(cos_in->layout.shape[0] >= most, WGF_ERR_SHAPE,
                  "cos / sin end at position " + std::to_string(cos_in->layout.shape[0]) + ", the append at " + std::to_string(most));
        out.dtype = c.dtype;
        out.layout = Layout::contiguous(qs);
    }
    dev.make_current();
    if (q_in) out.buf = dev.alloc((size_t)std::max<int64_t>(out.layout.numel(), 1) * dtype_size(c.dtype), most == 0);
    if (most == 0) return out;     // no sequence has or takes a token: q is padding, and cos / sin may be empty
    if (t == 0) return out;
    auto last_dense = [&](const TensorData& x) {
        const int l = x.layout.rank() - 1;
        return x.layout.strides[l] == 1 || x.layout.shape[l] == 1 ? x : run_compact(dev, x);
    };
    const TensorData k = last_dense(k_in), v = last_dense(v_in);
    TensorData q, wq, wk, cos, sin;
    AppendParams p{};
    unsigned q_ctas = 0;
    RowSpread s = head_spread(c.dtype, c.dim, {k.base_ptr(), v.base_ptr(), c.tail->ptr},
                              {k.layout.strides[0], k.layout.strides[1], k.layout.strides[2], v.layout.strides[0], v.layout.strides[1], v.layout.strides[2]});
    if (q_in) {
        q = last_dense(*q_in), wq = last_dense(*wq_in), wk = last_dense(*wk_in), cos = last_dense(*cos_in), sin = last_dense(*sin_in);
        for (const TensorData* x : {&q, &wq, &wk, &cos, &sin}) dev.wait_for(*x->buf);
        const RowSpread s2 = head_spread(c.dtype, c.dim, {q.base_ptr(), wq.base_ptr(), wk.base_ptr(), cos.base_ptr(), sin.base_ptr(), out.buf->ptr},
                                         {q.layout.strides[0], q.layout.strides[1], q.layout.strides[2], cos.layout.strides[0], sin.layout.strides[0]});
        if (s2.vec < s.vec) s = s2;
        p.q = q.base_ptr();
        p.wq = wq.base_ptr();
        p.wk = wk.base_ptr();
        p.cos = cos.base_ptr();
        p.sin = sin.base_ptr();
        p.q_out = out.buf->ptr;
        p.qb = q.layout.strides[0];
        p.qh = q.layout.strides[1];
        p.qs = q.layout.strides[2];
        p.cs_c = cos.layout.strides[0];
        p.cs_s = sin.layout.strides[0];
        p.q_heads = (int)q.layout.shape[1];
        p.table_rows = (int)std::min<int64_t>(cos.layout.shape[0], INT32_MAX);
        p.eps = eps;
        const int64_t rows = c.batch * q.layout.shape[1] * t, per = kThreads / s.lanes;
        WGF_CHECK(rows / per < (1ll << 30), WGF_ERR_UNSUPPORTED, "append of too many query rows in one call");
        q_ctas = (unsigned)((rows + per - 1) / per);
    }
    for (const TensorData* x : {&k, &v}) dev.wait_for(*x->buf);
    note(c);
    p.use_counts = !counts ? 0 : c.batch <= kGiven ? 2 : 1;
    if (p.use_counts == 1) kv_cache_set_counts(c, counts, t, "append");
    if (p.use_counts == 2) std::copy(counts, counts + c.batch, p.given);
    p.c = view_of(c);
    p.k = k.base_ptr();
    p.v = v.base_ptr();
    p.kb = k.layout.strides[0];
    p.kh = k.layout.strides[1];
    p.ks = k.layout.strides[2];
    p.vb = v.layout.strides[0];
    p.vh = v.layout.strides[1];
    p.vs = v.layout.strides[2];
    p.t = (int)t;
    p.blocks_touched = (int)((t + kBlock - 2) / kBlock + 1);
    run_append(dev, c, p, s, q_ctas, q_in != nullptr, q_in ? "kv_append_qk" : "kv_append");
    if (dev.recording()) {
        CacheStep* step = recorded_step(c);
        if (!step) {
            auto fresh = std::make_shared<CacheStep>();
            fresh->cache = c.shared_from_this();
            step = fresh.get();
            dev.recorded_steps().push_back(fresh);
        }
        step->added += t;
        if (q_in) step->table_rows = std::min(step->table_rows, cos_in->layout.shape[0]);
    } else {
        for (int64_t b = 0; b < c.batch; ++b) {
            c.lengths[b] += counts ? counts[b] : t;
            c.held_from[b] = std::max(c.held_from[b], c.lengths[b] / kBlock - 1);
        }
    }
    return out;
}

}  // namespace

int64_t KvCache::longest() const { return *std::max_element(lengths.begin(), lengths.end()); }
int64_t KvCache::recorded_tokens() const {
    const CacheStep* s = dev->recording() ? recorded_step(*this) : nullptr;
    return s ? s->added : 0;
}

KvCacheRef kv_cache_create(const DeviceRef& devref, DType dtype, int64_t batch, int64_t heads, int64_t dim, int64_t capacity) {
    Device& dev = *devref;
    dev.refuse_while_recording("making a cache");
    WGF_CHECK(batch >= 1 && heads >= 1 && capacity >= 1, WGF_ERR_SHAPE, "a cache needs at least one sequence, one head and room for one token");
    WGF_CHECK(dim >= 8 && dim <= 256 && dim % 8 == 0, WGF_ERR_UNSUPPORTED, "a cache's head_dim must be a multiple of 8 up to 256");
    WGF_CHECK(batch < (1 << 24) && heads < (1 << 24) && batch * heads < (1 << 28) && capacity < (1ll << 30), WGF_ERR_UNSUPPORTED, "cache extents too large");
    auto c = std::make_shared<KvCache>();
    c->dev = devref;
    c->dtype = dtype;
    c->batch = batch;
    c->heads = heads;
    c->dim = dim;
    c->dim_pad = (dim + 63) / 64 * 64;
    c->capacity = capacity;
    c->blocks = (capacity + KvCache::kBlock - 1) / KvCache::kBlock;
    WGF_CHECK(batch * heads < (1ll << 46) / (c->blocks * 2 * KvCache::kBlock * c->dim_pad), WGF_ERR_OOM, "the cache does not fit in memory");
    dev.make_current();
    const size_t bh = (size_t)(batch * heads);
    c->codes = dev.alloc(bh * c->blocks * 2 * KvCache::kBlock * c->dim_pad, false);
    c->scales = dev.alloc(bh * c->blocks * 2 * sizeof(float), false);
    c->tail = dev.alloc(bh * 2 * 2 * KvCache::kBlock * dim * dtype_size(dtype), false);
    c->lens = dev.alloc((size_t)batch * 2 * sizeof(int), true);
    c->lengths.assign(batch, 0);
    c->held_from.assign(batch, 0);
    return c;
}

void kv_cache_set_counts(KvCache& c, const int64_t* counts, int64_t t, const char* what) {
    if (c.dev->recording()) fail(WGF_ERR_UNSUPPORTED, std::string("counts of an ") + what + " are fixed numbers: a recording takes none");
    std::vector<int> v(c.batch);
    for (int64_t b = 0; b < c.batch; ++b) {
        WGF_CHECK(counts[b] >= 0 && counts[b] <= t, WGF_ERR_INVALID_ARGUMENT, "a count is not between 0 and the number of tokens given");
        v[b] = (int)counts[b];
    }
    set_ints(*c.dev, (int*)c.lens->ptr + c.batch, v, "kv_counts");
}

void kv_cache_truncate(KvCache& c, const int64_t* lengths) {
    Device& dev = *c.dev;
    dev.refuse_while_recording("truncating a cache");
    bool recode = false;
    std::vector<int> touched(c.batch, 0), lens(c.batch);
    for (int64_t b = 0; b < c.batch; ++b) {
        const int64_t n = lengths[b], blk = n / kBlock;
        WGF_CHECK(n >= 0 && n <= c.lengths[b], WGF_ERR_INVALID_ARGUMENT, "truncate cannot lengthen a sequence");
        WGF_CHECK(n == c.lengths[b] || n % kBlock == 0 || blk >= c.held_from[b], WGF_ERR_UNSUPPORTED,
                  "the tokens before " + std::to_string(c.held_from[b] * kBlock) + " of sequence " + std::to_string(b) +
                      " are held in 8 bits alone: truncate to a multiple of " + std::to_string(kBlock) + " there");
        lens[b] = (int)n;
        touched[b] = n != c.lengths[b] && n % kBlock != 0;
        recode = recode || touched[b];
    }
    dev.make_current();
    AppendParams p{};
    p.c = view_of(c);
    p.t = -1;
    p.blocks_touched = 1;
    const bool by_value = recode && c.batch <= kGiven;
    if (by_value) {
        p.use_counts = 2;
        for (int64_t b = 0; b < c.batch; ++b) p.given[b] = lens[b] | (touched[b] ? kRecode : 0);
    } else {
        set_ints(dev, (int*)c.lens->ptr, lens, "kv_truncate");
        if (recode) set_ints(dev, (int*)c.lens->ptr + c.batch, touched, "kv_counts");
        p.use_counts = 1;
    }
    if (recode) run_append(dev, c, p, head_spread(c.dtype, c.dim, {c.tail->ptr}, {}), 0, false, "kv_recode");
    for (int64_t b = 0; b < c.batch; ++b) {
        c.lengths[b] = lengths[b];
        c.held_from[b] = std::min(c.held_from[b], lengths[b] / kBlock);
    }
}

void kv_cache_append(KvCache& c, const TensorData& k, const TensorData& v, const int64_t* counts) {
    append(c, k, v, counts, nullptr, nullptr, nullptr, nullptr, nullptr, 0.f);
}

TensorData kv_cache_append_qk(KvCache& c, const TensorData& q, const TensorData& k, const TensorData& v, const TensorData& wq,
                              const TensorData& wk, const TensorData& cos, const TensorData& sin, float eps, const int64_t* counts) {
    return append(c, k, v, counts, &q, &wq, &wk, &cos, &sin, eps);
}

void kv_cache_read(KvCache& c, TensorData& k, TensorData& v) {
    Device& dev = *c.dev;
    dev.refuse_while_recording("reading a cache, whose length is part of the result's shape,");
    dev.make_current();
    const int64_t n = c.longest();
    for (TensorData* t : {&k, &v}) {
        t->dtype = c.dtype;
        t->layout = Layout::contiguous({c.batch, c.heads, n, c.dim});
        t->buf = dev.alloc((size_t)std::max<int64_t>(t->layout.numel(), 1) * dtype_size(c.dtype), false);
    }
    if (n == 0) return;
    const int64_t out_blocks = (n + kBlock - 1) / kBlock, ctas = 2 * c.batch * c.heads * out_blocks;
    WGF_CHECK(ctas < (1ll << 31), WGF_ERR_UNSUPPORTED, "read of more than 2^30 blocks in one call");
    auto go = [&](auto kernel, auto* ko, auto* vo) {
        dev.begin_launch("kv_read");
        if (!dev.dry) kernel<<<(unsigned)ctas, kThreads, 0, dev.stream>>>(view_of(c), ko, vo, (int)n, (int)out_blocks);
        dev.end_launch();
    };
    for_pad(c.dim_pad, [&](auto pad) {
        constexpr int DP = decltype(pad)::value;
        if (c.dtype == DType::F32) go(kv_read_kernel<float, DP>, (float*)k.buf->ptr, (float*)v.buf->ptr);
        else if (c.dtype == DType::F16) go(kv_read_kernel<__half, DP>, (__half*)k.buf->ptr, (__half*)v.buf->ptr);
        else go(kv_read_kernel<__nv_bfloat16, DP>, (__nv_bfloat16*)k.buf->ptr, (__nv_bfloat16*)v.buf->ptr);
    });
}

}  // namespace wgf
