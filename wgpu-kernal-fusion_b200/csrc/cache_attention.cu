// Attention of a few new tokens over the 8-bit cache, in one launch.
//
// For a row (query head and token) with the limit n of keys that it may see:
//   s_j = scale * q . K_j,  o = sum_j exp(s_j - max s) V_j / sum_j exp(s_j - max s),  j < n;   zeros for n = 0.
//
// What bounds it: every key and value of the cache is read once, 2 * head_dim bytes a token and kv head, for at most
// a few rows, so it is memory.  The product is done by the warps' own m16n8k16 instructions: their B operand comes
// from registers, which is where the codes are after the conversion to f16, while the fifth-generation instructions
// would want the converted operand in shared memory, twice the cache's bytes written and read there.
//   * A warp works on a block of 64 tokens by itself: running maximum, sum and accumulator in registers, no
//     barrier anywhere in the loop.  The cache is stored in the order in which lanes want it (kv_cache.cu), so a lane
//     copies the bytes that it will read itself (16 at a time, asynchronously, three half blocks in flight).
//   * Codes become f16 exactly: the byte is put under the exponent of 1024 and 1152 is taken off.
//   * The 16 rows of the instruction are 8 query rows twice: the f16 nearest to the value and the f16 nearest to what
//     that leaves.  Queries (scaled by a power of two of their own) and probabilities so keep 22 bits, for all element
//     types alike, at no cost: eight rows are as many as grouped heads commonly have.
//   * The lane that holds the scores of a row's tokens is the lane that needs them as the A operand of the second
//     product, because tokens are numbered so (key_token in kv_cache.cu): nothing is exchanged between the products.
//   * A sequence's blocks are split over CTAs when there are few heads, and over the four warps of a CTA; the
//     last CTA to finish a row tile joins the parts in their order, so results do not depend on timing.
#include <algorithm>

#include "decode.hpp"
#include "decode_common.cuh"

namespace wgf {

using namespace decode;

namespace {

constexpr int kBlock = KvCache::kBlock;
constexpr int kWarps = 4;
constexpr int kRows = 8;        // query rows of a tile
constexpr int kStages = 3;      // half blocks (keys or values of 64 tokens) in a warp's ring

struct AttParams {
    const uint8_t* codes;
    const float* scales;
    const int* lens;
    const void* q;
    void* out;
    long long qb, qh, qs;
    float* part;           // [job][split]{ [8] maxima, [8] sums, [8][dim_pad] }
    unsigned* tickets;     // [job]
    int batch, heads, blocks, dim, q_heads, group, t, use_counts;
    int rows, tiles;       // rows of a kv head, tiles of eight of them
    int splits, part_min;  // CTAs of a tile, and the blocks that one takes at least
    float scale_log2;
};

__device__ __forceinline__ unsigned pair_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ void split_f16(float a, float b, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const unsigned*>(&h);
    const float2 f = __half22float2(h);
    lo = pair_f16(a - f.x, b - f.y);
}
// Four codes (bytes, 128 added) as two pairs of f16
__device__ __forceinline__ void unpack(unsigned w, unsigned& a, unsigned& b) {
    const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
    const unsigned x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), off), q = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
    a = *reinterpret_cast<const unsigned*>(&p);
    b = *reinterpret_cast<const unsigned*>(&q);
}
__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shared memory of a CTA: the warps' rings, then the queries as A operands:
// [dims / 64][half of the chunk's four steps][lane] { step: a0 hi, a1 lo, a2 hi, a3 lo } x 2, and per row the power of
// two that its queries were scaled by.
template <int DP> constexpr size_t ring_bytes() { return (size_t)kWarps * kStages * kBlock * DP; }
template <int DP> constexpr size_t att_smem() { return ring_bytes<DP>() + (size_t)DP / 64 * 4 * 512 + kRows * 8; }

template <typename T, int DP>
__global__ void __launch_bounds__(kWarps * 32) cache_attention_kernel(const __grid_constant__ AttParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ unsigned last;
    constexpr int NJ = DP / 64;      // chunks of 64 dims
    constexpr int ND = DP / 8;       // groups of 8 dims
    const int split = blockIdx.x % p.splits;
    const int job = blockIdx.x / p.splits;
    const int tile = job % p.tiles, bh = job / p.tiles;
    const int h = bh % p.heads, b = bh / p.heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;

    const int len = p.lens[b];
    const int count = p.use_counts ? p.lens[p.batch + b] : p.t;
    // how many keys a row may see: those up to its own position
    auto limit = [&](int row) {
        const int i = row % p.t;
        return row < p.rows && i < count ? max(len - count + i + 1, 0) : 0;
    };
    int longest = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) longest = max(longest, limit(tile * kRows + r));
    const int nblk = (longest + kBlock - 1) / kBlock;
    const int part = max(p.part_min, (nblk + p.splits - 1) / p.splits);
    const int used = max((nblk + part - 1) / part, 1);           // CTAs with work; one writes the zeros of an empty tile
    if (split >= used) return;
    const int begin = split * part, end = min(nblk, begin + part);

    const uint8_t* base = p.codes + (long long)bh * p.blocks * (2ll * kBlock * DP);
    unsigned char* ring = smem + warp * (kStages * kBlock * DP) + lane * 16;
    // half block n of this warp: block begin + warp + (n / 2) * 4, keys (n even) or values
    const int mine = begin + warp < end ? (end - begin - warp + kWarps - 1) / kWarps : 0;
    auto fetch = [&](int n) {
        if (n < 2 * mine) {
            const uint8_t* src = base + ((long long)(begin + warp + (n >> 1) * kWarps) * 2 + (n & 1)) * (kBlock * DP) + lane * 16;
            unsigned char* dst = ring + (n % kStages) * (kBlock * DP);
#pragma unroll
            for (int i = 0; i < ND; ++i) copy16(dst + i * 512, src + i * 512);
        }
        copies_commit();
    };
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) fetch(n);

    // The queries, two rows a warp: largest magnitude, scaling by a power of two to about 2^13, split into two f16
    unsigned* qs = reinterpret_cast<unsigned*>(smem + ring_bytes<DP>());
    float* unscale = reinterpret_cast<float*>(qs + NJ * 4 * 128);
#pragma unroll
    for (int rr = 0; rr < kRows / kWarps; ++rr) {
        const int r = warp * (kRows / kWarps) + rr, row = tile * kRows + r;
        const bool live = limit(row) > 0;
        const int rc = min(row, p.rows - 1);
        const T* src = (const T*)p.q + b * p.qb + (long long)(h * p.group + rc / p.t) * p.qh + (rc % p.t) * p.qs;
        float x[DP / 32];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < DP / 64; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = i * 64 + lane * 2 + e;
                const float v = live && d < p.dim ? to_f<T>(src[d]) : 0.f;
                x[i * 2 + e] = v;
                top = max(top, abs_bits(v));
            }
        top = __reduce_max_sync(0xffffffffu, top);
        // exponent of the largest, kept where the scaling and its inverse are both ordinary numbers
        const int e2 = min(max((int)(top >> 23) - 127, -100), 127);
        const float up = __uint_as_float((unsigned)(127 + 13 - e2) << 23);
        if (lane == 0) unscale[r] = __uint_as_float((unsigned)(127 - 13 + e2) << 23) * p.scale_log2;
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) {
            unsigned hi, lo;
            split_f16(x[i * 2] * up, x[i * 2 + 1] * up, hi, lo);
            // dims d, d + 1 of chunk i: lane group d / 16, step (d % 16) / 4, register a0 / a2 by (d % 4) / 2
            const int d = lane * 2, cc = d >> 4, s = (d & 15) >> 2, second = (d & 3) >> 1;
            unsigned* to = qs + ((i * 4 + s) * 32 + r * 4 + cc) * 4 + second * 2;
            to[0] = hi;
            to[1] = lo;
        }
    }
    __syncthreads();

    float m = -INFINITY, l = 0.f, o[ND][2];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = 0.f;
    const int lim = limit(tile * kRows + g);
    const float mul = unscale[g];

    const float2* scales = reinterpret_cast<const float2*>(p.scales) + (long long)bh * p.blocks + begin + warp;
    float2 ahead = mine > 0 ? scales[0] : make_float2(0.f, 0.f);
    for (int it = 0; it < mine; ++it) {
        const int blk = begin + warp + it * kWarps;
        const float2 sc = ahead;
        if (it + 1 < mine) ahead = scales[(it + 1) * kWarps];
        copies_wait<kStages - 2>();
        const unsigned char* kb = ring + ((2 * it) % kStages) * (kBlock * DP);
        float s[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            uint4 a[4];
#pragma unroll
            for (int st = 0; st < 4; ++st) a[st] = *reinterpret_cast<const uint4*>(qs + ((j * 4 + st) * 32 + lane) * 4);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint4 w = *reinterpret_cast<const uint4*>(kb + (n * NJ + j) * 512);
                const unsigned ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    unsigned b0, b1;
                    unpack(ws[st], b0, b1);
                    mma(s[n], a[st].x, a[st].y, a[st].z, a[st].w, b0, b1);
                }
            }
        }
        fetch(2 * it + kStages - 1);

        // scores of row g, tokens 16 c + 4 (n / 2) + 2 (n % 2) + e of the block
        const float ks = sc.x * mul;
        const int room = lim - blk * kBlock;               // tokens of this block that the row sees
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int token = c * 16 + (n >> 1) * 4 + (n & 1) * 2 + e;
                const float v = token < room ? (s[n][e] + s[n][2 + e]) * ks : -INFINITY;
                s[n][e] = v;
                top = fmaxf(top, v);
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m2 = fmaxf(m, top);
        const float from = m2 == -INFINITY ? 0.f : m2;     // nothing seen yet: every probability below is 0
        const float keep = exp2f(m - from);
        m = m2;
        float sum = 0.f;
        unsigned ph[8], pl[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float p0 = exp2f(s[n][0] - from), p1 = exp2f(s[n][1] - from);
            sum += p0 + p1;
            split_f16(p0, p1, ph[n], pl[n]);
        }
        l = l * keep + sum;                                // this lane's tokens; the four lanes are added at the end

        copies_wait<kStages - 2>();
        const unsigned char* vb = ring + ((2 * it + 1) % kStages) * (kBlock * DP);
        const float vs = room > 0 ? sc.y : 0.f;            // a row that sees nothing of the block takes nothing of its scale
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(vb + i * 512);
            const unsigned ws[4] = {w.x, w.y, w.z, w.w};
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                unsigned b0, b1;
                unpack(ws[st], b0, b1);
                mma(acc, ph[2 * st], pl[2 * st], ph[2 * st + 1], pl[2 * st + 1], b0, b1);
            }
            o[i][0] = o[i][0] * keep + (acc[0] + acc[2]) * vs;
            o[i][1] = o[i][1] * keep + (acc[1] + acc[3]) * vs;
        }
        fetch(2 * it + kStages);
    }
    copies_wait<0>();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // The warps' parts through shared memory: [warp][row]{maximum, sum}, [warp][row][dim]
    __syncthreads();                                       // the rings are free
    float* wm = reinterpret_cast<float*>(smem);
    float* wl = wm + kWarps * kRows;
    float* wo = wl + kWarps * kRows;
    if (c == 0) {
        wm[warp * kRows + g] = m;
        wl[warp * kRows + g] = l;
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) *reinterpret_cast<float2*>(wo + (warp * kRows + g) * DP + i * 8 + c * 2) = make_float2(o[i][0], o[i][1]);
    __syncthreads();
    const int live_rows = min(kRows, p.rows - tile * kRows);
    constexpr int kPart = 2 * kRows + kRows * DP;
    auto put = [&](int r, int d, float v) {
        const int row = tile * kRows + r;
        ((T*)p.out)[(((long long)b * p.q_heads + h * p.group) * p.t + row) * p.dim + d] = from_f<T>(v);
    };
    float* mypart = p.part + ((long long)job * p.splits + split) * kPart;
    for (int i = threadIdx.x; i < live_rows * DP; i += kWarps * 32) {
        const int r = i / DP, d = i - r * DP;
        float top = wm[r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, wm[w * kRows + r]);
        const float from = top == -INFINITY ? 0.f : top;
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(wm[w * kRows + r] - from);
            sum += wl[w * kRows + r] * f;
            acc += wo[(w * kRows + r) * DP + d] * f;
        }
        if (used == 1) {
            if (d < p.dim) put(r, d, sum == 0.f ? 0.f : acc / sum);
        } else {
            mypart[2 * kRows + i] = acc;
            if (d == 0) {
                mypart[r] = top;
                mypart[kRows + r] = sum;
            }
        }
    }
    if (used == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.tickets + job, 1u) == (unsigned)used - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    const float* parts = p.part + (long long)job * p.splits * kPart;
    for (int i = threadIdx.x; i < live_rows * DP; i += kWarps * 32) {
        const int r = i / DP, d = i - r * DP;
        float top = -INFINITY;
        for (int n = 0; n < used; ++n) top = fmaxf(top, __ldcg(parts + (long long)n * kPart + r));
        const float from = top == -INFINITY ? 0.f : top;
        float sum = 0.f, acc = 0.f;
        for (int n = 0; n < used; ++n) {
            const float* q = parts + (long long)n * kPart;
            const float f = exp2f(__ldcg(q + r) - from);
            sum += __ldcg(q + kRows + r) * f;
            acc += __ldcg(q + 2 * kRows + i) * f;
        }
        if (d < p.dim) put(r, d, sum == 0.f ? 0.f : acc / sum);
    }
    if (threadIdx.x == 0) p.tickets[job] = 0;
}

template <typename T, int DP> void launch_att(Device& dev, const AttParams& p, unsigned grid) {
    auto kernel = cache_attention_kernel<T, DP>;
    constexpr size_t smem = att_smem<DP>();
    if (!dev.dry) {
        static unsigned long long done = 0;    // one bit a device; setting it twice does no harm
        if (dev.ordinal >= 64 || !(done >> dev.ordinal & 1)) {
            WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            if (dev.ordinal < 64) done |= 1ull << dev.ordinal;
        }
    }
    dev.begin_launch("cache_attention");
    if (!dev.dry) kernel<<<grid, kWarps * 32, smem, dev.stream>>>(p);
    dev.end_launch();
}

template <typename T> void dispatch_att(Device& dev, const AttParams& p, unsigned grid, int64_t dp) {
    switch (dp) {
        case 64: return launch_att<T, 64>(dev, p, grid);
        case 128: return launch_att<T, 128>(dev, p, grid);
        case 192: return launch_att<T, 192>(dev, p, grid);
        default: return launch_att<T, 256>(dev, p, grid);
    }
}

}  // namespace

TensorData kv_cache_attention(KvCache& c, const TensorData& q_in, float scale, const int64_t* counts) {
    Device& dev = *c.dev;
    WGF_CHECK(q_in.layout.rank() == 4, WGF_ERR_RANK, "queries must be [batch, query heads, tokens, head_dim]");
    WGF_CHECK(q_in.dtype == c.dtype, WGF_ERR_DTYPE, "queries differ from the cache in element type");
    const auto& s = q_in.layout.shape;
    WGF_CHECK(s[0] == c.batch && s[3] == c.dim && s[1] % c.heads == 0, WGF_ERR_SHAPE,
              "queries must be [" + std::to_string(c.batch) + ", a multiple of " + std::to_string(c.heads) + " heads, tokens, " + std::to_string(c.dim) + "]");
    const int64_t group = s[1] / c.heads, t = s[2];
    WGF_CHECK(group * t < (1ll << 30), WGF_ERR_UNSUPPORTED, "too many query rows");
    if (counts)
        for (int64_t b = 0; b < c.batch; ++b)
            WGF_CHECK(counts[b] >= 0 && counts[b] <= t, WGF_ERR_INVALID_ARGUMENT, "a count is not between 0 and the number of tokens given");
    dev.make_current();
    TensorData q = q_in.layout.strides[3] == 1 || c.dim == 1 ? q_in : run_compact(dev, q_in), out;
    dev.wait_for(*q.buf);
    out.dtype = c.dtype;
    out.layout = Layout::contiguous(s);
    out.buf = dev.alloc((size_t)std::max<int64_t>(out.layout.numel(), 1) * dtype_size(c.dtype), false);
    if (out.layout.numel() == 0) return out;
    for (const BufferRef& b : {c.codes, c.scales, c.tail, c.lens}) dev.note_recorded_buffer(b);
    if (counts) kv_cache_set_counts(c, counts, t, "attention");
    AttParams p{};
    p.codes = (const uint8_t*)c.codes->ptr;
    p.scales = (const float*)c.scales->ptr;
    p.lens = (const int*)c.lens->ptr;
    p.q = q.base_ptr();
    p.out = out.buf->ptr;
    p.qb = q.layout.strides[0];
    p.qh = q.layout.strides[1];
    p.qs = q.layout.strides[2];
    p.batch = (int)c.batch;
    p.heads = (int)c.heads;
    p.blocks = (int)c.blocks;
    p.dim = (int)c.dim;
    p.q_heads = (int)s[1];
    p.group = (int)group;
    p.t = (int)t;
    p.use_counts = counts != nullptr;
    p.rows = (int)(group * t);
    p.tiles = (p.rows + kRows - 1) / kRows;
    p.scale_log2 = scale * 1.4426950408889634f;
    // How the blocks are split.  CTAs of a tile are wanted until the GPU is full, but none with fewer blocks than
    // warps.  A recording stays right while the cache grows, so it plans for the longest that a sequence can get.
    const int64_t jobs = c.batch * c.heads * p.tiles;
    int64_t most = 0, total = 0;
    for (int64_t b = 0; b < c.batch; ++b) {
        const int64_t n = ((dev.recording() ? c.capacity : c.lengths[b]) + kBlock - 1) / kBlock;
        most = std::max(most, n);
        total += n;
    }
    total *= c.heads * p.tiles;
    const int64_t per_sm = std::max<int64_t>(1, (int64_t)(227 * 1024) / (int64_t)(kWarps * kStages * kBlock * c.dim_pad + c.dim_pad * 32 + 2048));
    const int64_t slots = dev.sm_count * std::min<int64_t>(per_sm, 4);
    p.splits = 1;
    p.part_min = (int)std::max<int64_t>(most, 1);
    if (jobs <= Device::kCounters && most > kWarps) {
        const int64_t part = std::max<int64_t>(kWarps, (total + slots - 1) / slots);
        p.splits = (int)std::min<int64_t>((most + part - 1) / part, 1024);
        p.part_min = dev.recording() ? kWarps : (int)std::max<int64_t>(part, (most + p.splits - 1) / p.splits);
    }
    BufferRef scratch;
    if (p.splits > 1) {
        scratch = dev.alloc((size_t)(jobs * p.splits) * (2 * kRows + kRows * c.dim_pad) * sizeof(float), false);
        p.part = (float*)scratch->ptr;
        p.tickets = (unsigned*)dev.counters();
    }
    WGF_CHECK(jobs * p.splits < (1ll << 31), WGF_ERR_UNSUPPORTED, "attention over too many heads and rows in one call");
    const unsigned grid = (unsigned)(jobs * p.splits);
    if (c.dtype == DType::F32) dispatch_att<float>(dev, p, grid, c.dim_pad);
    else if (c.dtype == DType::F16) dispatch_att<__half>(dev, p, grid, c.dim_pad);
    else dispatch_att<__nv_bfloat16>(dev, p, grid, c.dim_pad);
    return out;
}

}  // namespace wgf
