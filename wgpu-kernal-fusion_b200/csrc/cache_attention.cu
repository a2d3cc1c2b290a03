// Attention of a few new tokens over the 8-bit cache, in one launch.
//
// For a row (query head and token) with the limit n of keys that it may see:
//   s_j = scale * q . K_j,  o = sum_j exp(s_j - max s) V_j / sum_j exp(s_j - max s),  j < n;   zeros for n = 0.
//
// What bounds it: every key and value of the cache is read once, 2 * head_dim bytes a token and kv head, for at most
// a few rows, so it is memory.  The product is done by the warps' own m16n8k16 instructions: their B operand comes
// from registers, which is where the codes are after the conversion to f16.  The fifth-generation instructions take operands from
// shared and tensor memory, where every converted code would have to be written first, for eight rows that use it.
//   * A warp works on a block of 64 tokens by itself: running maximum, sum and accumulator in registers, no
//     barrier anywhere in the loop.  The cache is stored in the order in which lanes want it (kv_cache.cu), so a lane
//     copies the bytes that it will read itself (16 at a time, asynchronously, three half blocks in flight).
//   * Codes become f16 exactly: the byte is put under the exponent of 1024 and 1152 is taken off.
//   * The 16 rows of the instruction are 8 query rows twice: the f16 nearest to the value and the f16 nearest to what
//     that leaves.  Both kinds are first brought to the upper end of the type's range, queries by a power of two of their own,
//     probabilities by 2^15: what the two f16 lose is 2^-22 of a value, or 2^-38 of the row's largest one where that is more.  So many
//     small probabilities beside a dominant one keep their digits, for all element types alike, at no cost: eight rows are as
//     many as grouped heads commonly have.
//   * The lane that holds the scores of a row's tokens is the lane that needs them as the A operand of the second
//     product, because tokens are numbered so (key_token in kv_cache.cu): nothing is exchanged between the products.
//   * The work of all sequences, heads and row tiles is laid end to end in units of four blocks (one for each warp of
//     a CTA), and every CTA takes an equal stretch of it, as the kernel itself computes from the lengths: ragged
//     batches are even, and a recorded launch stays even while its sequences grow.  The last CTA to finish a job
//     that several have a stretch of joins their parts, in their order, so results do not depend on timing.
// One token over 131071 of 8 kv heads, 269 MB: the CTAs' loops take 42 us (6.4 TB/s of the measured 6.56), a pass 55 to 57 us by card with
// the launch, the first loads and the joining; with two half blocks in a ring instead of three it took 87.  32 sequences of up to
// 8192 tokens, 310 MB: 74 to 76 us, 84 where each job had a number of CTAs of its own.
#include <algorithm>

#include "decode.hpp"
#include "decode_common.cuh"

namespace wgf {

using namespace decode;

namespace {

constexpr int kBlock = KvCache::kBlock;
constexpr int kWarps = 4;
constexpr int kGiven = 256;
constexpr int kRows = 8;        // query rows of a tile
constexpr int kMaxBatch = 1024; // sequences whose work is shared out evenly
constexpr int kStages = 3;      // half blocks (keys or values of 64 tokens) in a warp's ring
constexpr float kProbUp = 32768.f;   // probabilities, at most 1, go to the upper end of f16 before they are split

struct AttParams {
    const uint8_t* codes;
    const float* scales;
    const int* lens;
    const void* q;
    void* out;
    long long qb, qh, qs;
    float* part;           // [CTA][first or last stretch]{ [8] maxima, [8] sums, [8][dim_pad] }
    unsigned* tickets;     // [job]
    int batch, heads, blocks, dim, q_heads, group, t, use_counts;
    int rows, tiles;       // rows of a kv head, tiles of eight of them
    int whole;             // one CTA for each job
    float scale_log2;
    int given[kGiven];     // counts of a small batch (use_counts == 2; 1: in the second half of lens)
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
// Shared memory of a CTA: the warps' rings, then the queries as A operands:
// [dims / 64][half of the chunk's four steps][lane] { step: a0 hi, a1 lo, a2 hi, a3 lo } x 2, and per row the power of
// two that its queries were scaled by.
template <int DP> constexpr size_t ring_bytes() { return (size_t)kWarps * kStages * kBlock * DP; }
template <int DP> constexpr size_t att_smem() { return ring_bytes<DP>() + (size_t)DP / 64 * 4 * 512 + kRows * 8; }

// Quads (four blocks, one for each warp) of a sequence; at least one, for the zeros of an empty sequence
__device__ __forceinline__ int quads_of(const AttParams& p, int b) { return max((p.lens[b] + kWarps * kBlock - 1) / (kWarps * kBlock), 1); }

// Fills before[0 .. batch] with running sums of the sequences' quads in pieces of `share` and returns the last.
__device__ __forceinline__ int scan_quads(const AttParams& p, int* before, int share) {
    __shared__ int sums[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kWarps * 32) {
        const int b = b0 + threadIdx.x;
        int x = b < p.batch ? (quads_of(p, b) + share - 1) / share : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        for (int w = 0; w < warp; ++w) x += sums[w];
        if (b < p.batch) before[b + 1] = run + x;
        for (int w = 0; w < kWarps; ++w) run += sums[w];
        __syncthreads();
    }
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    return run;
}
// How many pieces of `share` quads all sequences have; every warp adds them up for itself.
__device__ __forceinline__ int pieces_of(const AttParams& p, const int* before, int share) {
    int n = 0;
    for (int b = threadIdx.x & 31; b < p.batch; b += 32) n += (before[b + 1] - before[b] + share - 1) / share;
    return __reduce_add_sync(0xffffffffu, n);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kWarps * 32) cache_attention_kernel(const __grid_constant__ AttParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ unsigned last;
    __shared__ float total[kRows];
    __shared__ int before[kMaxBatch + 1];                        // quads, or pieces, of a head's tile in the sequences before
    constexpr int NJ = DP / 64;      // chunks of 64 dims
    constexpr int ND = DP / 8;       // groups of 8 dims
    constexpr int kPart = 2 * kRows + kRows * DP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    unsigned char* ring = smem + warp * (kStages * kBlock * DP) + lane * 16;
    const long long ht = (long long)p.heads * p.tiles;

    // This CTA's share of all quads: [at, stop).  A job's end within a share costs about as much as two quads, so where
    // there are enough CTAs for short shares that end with their jobs, and are at most two quads longer, they do (`pieces`:
    // `at` then counts pieces).  With `whole`, one job's.
    long long at = 0, stop = 1, share = 1;
    bool pieces = false;
    if (!p.whole) {
        const long long all = ht * scan_quads(p, before, 1);
        share = (all + gridDim.x - 1) / gridDim.x;
        for (int longer = 0; longer < 3 && !pieces && share > 1 && share <= 16; ++longer) pieces = ht * pieces_of(p, before, (int)share + longer) <= gridDim.x && (share += longer, true);
        if (pieces) {
            __syncthreads();
            const long long n = ht * scan_quads(p, before, (int)share);
            at = blockIdx.x;
            stop = min(n, at + 1);
        } else {
            at = (long long)blockIdx.x * share;
            stop = min(all, at + share);
        }
    }
    const long long first = at;
    while (at < stop) {
        int b;
        long long job_at, quads, hj;                                 // of the job at hand: its first quad, how many, head and tile
        if (p.whole) {
            b = (int)(blockIdx.x / ht);
            hj = blockIdx.x - b * ht;
            job_at = 0;
            quads = 1ll << 30;
        } else {
            int lo = 0, hi = p.batch - 1;                            // the last sequence that begins at or before `at`
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (before[mid] * ht <= at) lo = mid;
                else hi = mid - 1;
            }
            b = lo;
            quads = before[b + 1] - before[b];
            hj = (at - before[b] * ht) / quads;
            job_at = before[b] * ht + hj * quads;
        }
        const int h = (int)(hj / p.tiles), tile = (int)(hj - (long long)h * p.tiles);
        const long long bh = (long long)b * p.heads + h, job = b * ht + hj;
        const long long seg = p.whole ? quads : min(stop, job_at + quads) - at;
        const long long scale_up = pieces ? share : 1;               // quads of a unit of `at`
        const int len = p.lens[b];
        const int count = p.use_counts == 2 ? p.given[b] : p.use_counts ? p.lens[p.batch + b] : p.t;
        // how many keys a row may see: those up to its own position
        auto limit = [&](int row) {
            const int i = row % p.t;
            return row < p.rows && i < count ? max(len - count + i + 1, 0) : 0;
        };
        const int nblk = (len + kBlock - 1) / kBlock;
        const int begin = (int)min((at - job_at) * scale_up * kWarps, (long long)nblk), end = (int)min((at - job_at + seg) * scale_up * kWarps, (long long)nblk);

        const uint8_t* base = p.codes + bh * p.blocks * (2ll * kBlock * DP);
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

        const float2* scales = reinterpret_cast<const float2*>(p.scales) + bh * p.blocks + begin + warp;
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
                split_f16(p0 * kProbUp, p1 * kProbUp, ph[n], pl[n]);
            }
            l = l * keep + sum;                                // this lane's tokens; the four lanes are added at the end

            copies_wait<kStages - 2>();
            const unsigned char* vb = ring + ((2 * it + 1) % kStages) * (kBlock * DP);
            const float vs = room > 0 ? sc.y * (1.f / kProbUp) : 0.f;            // a row that sees nothing of the block takes nothing of its scale
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

        // The warps' parts through shared memory: [warp][row]{maximum, sum, weight}, [warp][row][dim]
        __syncthreads();                                       // the rings are free
        float* wm = reinterpret_cast<float*>(smem);
        float* wl = wm + kWarps * kRows;
        float* wf = wl + kWarps * kRows;
        float* wo = wf + kWarps * kRows;
        if (c == 0) {
            wm[warp * kRows + g] = m;
            wl[warp * kRows + g] = l;
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) *reinterpret_cast<float2*>(wo + (warp * kRows + g) * DP + i * 8 + c * 2) = make_float2(o[i][0], o[i][1]);
        __syncthreads();
        const int live_rows = min(kRows, p.rows - tile * kRows);
        // The CTAs that have a stretch of this job; a CTA's first stretch and its last one have places of their own.
        const long long per = pieces ? 1 : share;                    // units of `at` a CTA
        const long long cta0 = p.whole ? 0 : job_at / per, cta1 = p.whole ? 0 : (job_at + quads - 1) / per;
        const int used = (int)(cta1 - cta0) + 1;
        float* mypart = p.part + ((long long)blockIdx.x * 2 + (at != first)) * kPart;
        if (threadIdx.x < kRows) {
            const int r = threadIdx.x;
            float top = wm[r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, wm[w * kRows + r]);
            const float from = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2f(wm[w * kRows + r] - from);
                wf[w * kRows + r] = f;
                sum += wl[w * kRows + r] * f;
            }
            wl[r] = sum;
            if (used > 1) {
                mypart[r] = top;
                mypart[kRows + r] = sum;
            }
        }
        __syncthreads();
        T* out = (T*)p.out + (((long long)b * p.q_heads + h * p.group) * p.t + tile * kRows) * p.dim;
        // four dims of a row: what is left of the sums' weight is taken out, and they are rounded
        auto put = [&](int r, int d, float4 v, float sum) {
            const float x[4] = {v.x, v.y, v.z, v.w};
            Pack<T, 4> y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.v[e] = from_f<T>(sum == 0.f ? 0.f : x[e] / sum);
            if (d < p.dim) *reinterpret_cast<Pack<T, 4>*>(out + (long long)r * p.dim + d) = y;     // head_dim is a multiple of 8
        };
        for (int i = threadIdx.x * 4; i < live_rows * DP; i += kWarps * 32 * 4) {
            const int r = i / DP, d = i - r * DP;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = wf[w * kRows + r];
                const float4 v = *reinterpret_cast<const float4*>(wo + (w * kRows + r) * DP + d);
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (used == 1) put(r, d, acc, wl[r]);
            else *reinterpret_cast<float4*>(mypart + 2 * kRows + i) = acc;
        }
        if (used > 1) {
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();                               // behind the barrier: for all that the CTA has written
                last = atomicAdd(p.tickets + job, 1u) == (unsigned)used - 1;
                __threadfence();
            }
            __syncthreads();
            if (last) {
                // part n is the first stretch of its CTA, but for a job that begins in the middle of a CTA's share
                const float* parts = p.part + cta0 * 2 * kPart;
                const int shift = job_at > cta0 * per ? kPart : 0;
                // All the maxima and sums, and as many parts as shared memory takes, come in one go; a thread copies what it
                // will add up itself.
                float* ml = reinterpret_cast<float*>(smem);    // [part]{ [8] maxima, then weights; [8] sums }
                float* data = ml + used * 16;
                const int quarter = live_rows * DP / 4;        // 16-byte pieces of a part
                const int room = ((int)ring_bytes<DP>() - used * 64) / (quarter * 16);
                auto bring = [&](int n0) {
                    const int n1 = min(used, n0 + room);
                    for (int i = threadIdx.x; i < quarter; i += kWarps * 32) {
                        float* dst = data + i * 4;
                        const float* src = parts + (long long)n0 * 2 * kPart + 2 * kRows + i * 4;
                        int n = n0;
                        if (n == 0) {
                            copy16(dst, src + shift);
                            ++n, dst += quarter * 4, src += 2 * kPart;
                        }
#pragma unroll 4
                        for (; n < n1; ++n, dst += quarter * 4, src += 2 * kPart) copy16(dst, src);
                    }
                    copies_commit();
                };
                for (int i = threadIdx.x; i < used * 4; i += kWarps * 32) copy16(ml + i * 4, parts + (long long)(i >> 2) * 2 * kPart + (i < 4 ? shift : 0) + (i & 3) * 4);
                copies_commit();
                bring(0);
                copies_wait<0>();
                __syncthreads();
                for (int r = warp; r < live_rows; r += kWarps) {
                    float top = -INFINITY;
                    for (int n = lane; n < used; n += 32) top = fmaxf(top, ml[n * 16 + r]);
#pragma unroll
                    for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float from = top == -INFINITY ? 0.f : top;
                    float sum = 0.f;
                    for (int n = lane; n < used; n += 32) {
                        const float f = exp2f(ml[n * 16 + r] - from);
                        ml[n * 16 + r] = f;
                        sum += ml[n * 16 + kRows + r] * f;
                    }
#pragma unroll
                    for (int x = 16; x >= 1; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                    if (lane == 0) total[r] = sum;
                }
                __syncthreads();
                float4 acc[kRows * DP / (kWarps * 128)];
#pragma unroll
                for (int k = 0; k < kRows * DP / (kWarps * 128); ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int n0 = 0; n0 < used; n0 += room) {
                    if (n0 > 0) {
                        bring(n0);
                        copies_wait<0>();
                    }
#pragma unroll
                    for (int k = 0; k < kRows * DP / (kWarps * 128); ++k) {
                        const int i = threadIdx.x + k * kWarps * 32;
                        if (i >= quarter) break;
                        const int r = i * 4 / DP;
                        const int n1 = min(used, n0 + room);
                        const float* src = data + i * 4;
                        const float* weight = ml + n0 * 16 + r;
#pragma unroll 4
                        for (int n = n0; n < n1; ++n, src += quarter * 4, weight += 16) {
                            const float4 v = *reinterpret_cast<const float4*>(src);
                            const float f = *weight;
                            acc[k].x += v.x * f;
                            acc[k].y += v.y * f;
                            acc[k].z += v.z * f;
                            acc[k].w += v.w * f;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < kRows * DP / (kWarps * 128); ++k) {
                    const int i = threadIdx.x + k * kWarps * 32;
                    if (i < quarter) put(i * 4 / DP, i * 4 % DP, acc[k], total[i * 4 / DP]);
                }
                if (threadIdx.x == 0) p.tickets[job] = 0;
            }
        }
        at += seg;
        if (at < stop) __syncthreads();                        // the next job's copies go where this one's parts were
    }
}

template <typename T, int DP> void launch_att(Device& dev, const AttParams& p, unsigned grid) {
    auto kernel = cache_attention_kernel<T, DP>;
    constexpr size_t smem = att_smem<DP>();
    if (!dev.dry) {
        static unsigned long long done = 0;    // one bit a device; setting it twice does no harm
        if (dev.ordinal >= 64 || !(done >> dev.ordinal & 1)) {
            WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared));
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
    if (counts && dev.recording()) fail(WGF_ERR_UNSUPPORTED, "counts of an attention are fixed numbers: a recording takes none");
    AttParams p{};
    p.use_counts = !counts ? 0 : c.batch <= kGiven ? 2 : 1;
    if (p.use_counts == 1) kv_cache_set_counts(c, counts, t, "attention");
    if (p.use_counts == 2) std::copy(counts, counts + c.batch, p.given);
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
    p.rows = (int)(group * t);
    p.tiles = (p.rows + kRows - 1) / kRows;
    p.scale_log2 = scale * 1.4426950408889634f;
    // CTAs for the whole GPU; each takes an equal run of all the jobs' quads, job after job.  (A recording stays right while
    // the cache grows: it has CTAs for the longest that its sequences can get.)  Where there are more jobs than
    // tickets, or sequences than the kernel sums up, there is enough to do without dividing any.
    const int64_t jobs = c.batch * c.heads * p.tiles;
    p.whole = jobs > Device::kCounters || c.batch > kMaxBatch;
    int64_t quads = 0;
    for (int64_t b = 0; b < c.batch; ++b)
        quads += std::max<int64_t>(((dev.recording() ? c.capacity : c.lengths[b]) + kBlock * kWarps - 1) / (kBlock * kWarps), 1);
    quads *= c.heads * p.tiles;
    const int64_t per_sm = std::max<int64_t>(1, (int64_t)(227 * 1024) / (int64_t)(kWarps * kStages * kBlock * c.dim_pad + c.dim_pad * 32 + 6144));
    const int64_t ctas = p.whole ? jobs : std::min<int64_t>(quads, dev.sm_count * std::min<int64_t>(per_sm, 4));
    WGF_CHECK(ctas < (1ll << 31), WGF_ERR_UNSUPPORTED, "attention over too many heads and rows in one call");
    BufferRef scratch;
    if (!p.whole) {
        scratch = dev.alloc((size_t)(ctas * 2) * (2 * kRows + kRows * c.dim_pad) * sizeof(float), false);
        p.part = (float*)scratch->ptr;
        p.tickets = (unsigned*)dev.counters();
    }
    const unsigned grid = (unsigned)ctas;
    if (c.dtype == DType::F32) dispatch_att<float>(dev, p, grid, c.dim_pad);
    else if (c.dtype == DType::F16) dispatch_att<__half>(dev, p, grid, c.dim_pad);
    else dispatch_att<__nv_bfloat16>(dev, p, grid, c.dim_pad);
    return out;
}

}  // namespace wgf
