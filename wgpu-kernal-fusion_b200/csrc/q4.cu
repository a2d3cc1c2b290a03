// Products with 4-bit weights.
//
//   y[m, n] = sum over groups of columns of scale[n, group] * sum_{k in group} x[m, k] * (code[n, k] - 8)
//
// The weights are stored in tiles of 16 rows by 64 columns, 512 bytes, in the order in which the lanes of a warp want them
// as the A operand of four m16n8k16 instructions: lane (g, c) has 16 bytes, one word a step, with columns
// 32 (step / 2) + 8 c + 4 (step % 2) .. + 3 of rows g and g + 8, so that two steps are 32 columns in a row.  Within a word the two values that become one register are 16 bits apart:
//   nibble  0 / 4: row g, columns 0 / 1      1 / 5: row g + 8, columns 0 / 1
//           2 / 6: row g, columns 2 / 3      3 / 7: row g + 8, columns 2 / 3
// The scales of a tile's 16 rows stand side by side for each group.
//
// Few rows of x: every weight is read once, half a byte each, and used for at most a few multiplications, so memory is the bound.  The
// instruction's eight columns are the rows of x; codes become f16 or bf16 exactly (the nibble is put under the exponent of
// 1024 or 128, and 1032 or 136 is taken off; as bf16 they are 2^-10 of that until the end), and sums are f32 within a group and across groups.  A row of f32 takes three
// columns: its bf16 parts, which together have its 24 bits.  Operands go straight from global memory into
// registers; x is small and stays in the first-level cache.  The matrix does not go through tensor memory: for eight
// columns a tile of 128 rows would have to be converted into shared memory first, and the conversion, not the
// product, is the work here.
// Many rows: the weights are written out in the type of x once and the matrix product kernels take them.
#include <algorithm>

#include <cooperative_groups.h>

#include "decode.hpp"
#include "decode_common.cuh"

namespace wgf {

using namespace decode;
namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ float scale_at(const void* s, DType dt, long long i) {
    return dt == DType::F32 ? ((const float*)s)[i] : dt == DType::F16 ? __half2float(((const __half*)s)[i]) : __bfloat162float(((const __nv_bfloat16*)s)[i]);
}

// ---- making weights --------------------------------------------------------------------------------------------------
// Codes by value: scale = max|w| * (1/7), the product of two f32 numbers, rounded to the type of w; code = round(w / scale) + 8,
// ties to even, as if the quotient were exact.  One warp for rows g and g + 8 of a
// tile and one group; lane l has columns 4 l .. 4 l + 3 of the group.
template <typename T>
__global__ void q4_quantize_kernel(const T* __restrict__ w, long long rs, long long cs, uint32_t* __restrict__ codes, T* __restrict__ scales,
                                   long long n, long long k, int group, long long chunks, long long groups, long long padded, long long jobs) {
    const int lane = threadIdx.x & 31;
    for (long long job = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); job < jobs; job += (long long)gridDim.x * (blockDim.x >> 5)) {
        const int g = (int)(job & 7);
        const long long q = (job >> 3) % padded, rt = (job >> 3) / padded;
        const bool active = lane * 4 < group;
        unsigned nib[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const long long row = rt * 16 + g + half * 8;
            float x[4];
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const long long col = q * group + lane * 4 + e;
                x[e] = active && row < n && col < k ? to_f<T>(w[row * rs + col * cs]) : 0.f;
                top = max(top, abs_bits(x[e]));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const bool finite = top < 0x7f800000u;
            const T st = from_f<T>(finite ? __uint_as_float(top) * (1.f / 7.f) : __uint_as_float(0x7fc00000u));
            const float s = to_f<T>(st);
            const bool use = finite && s > 0.f;
            // far up and far down the quotient's sides are moved by a power of two that both can take
            const float move = s > 0x1p100f ? 0x1p-32f : s < 0x1p-90f ? 0x1p64f : 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                int code = 0;
                if (use) {
                    // a scale that was rounded down far (a type's smallest numbers) leaves quotients above 7
                    const float lim = 9.f * s;
                    code = exact_code(fminf(fmaxf(x[e], -lim), lim), move, s * move, 1.f / (s * move));
                }
                nib[half][e] = (unsigned)(min(max(code, -8), 7) + 8);
            }
            if (lane == 0 && q < groups) scales[(rt * groups + q) * 16 + g + half * 8] = st;
        }
        if (active) {
            const long long col = q * group + lane * 4, chunk = col / 64;
            const int c = (int)(col % 32) / 8, st = (int)(col % 64) / 32 * 2 + (int)(col % 8) / 4;
            const unsigned word = nib[0][0] | nib[1][0] << 4 | nib[0][2] << 8 | nib[1][2] << 12 | nib[0][1] << 16 | nib[1][1] << 20 |
                                  nib[0][3] << 24 | nib[1][3] << 28;
            if (chunk < chunks) codes[((rt * chunks + chunk) * 32 + g * 4 + c) * 4 + st] = word;
        }
    }
}

// Which nibble of a word belongs to row g + 8 * half, column e of its four
__device__ __forceinline__ int nibble(int half, int e) { return (e >> 1) * 2 + half + (e & 1) * 4; }

// Codes as a checkpoint has them: two columns a byte, the even one in the low half, rows one after the other.
__global__ void q4_pack_kernel(const uint8_t* __restrict__ in, uint32_t* __restrict__ codes, long long n, long long k, long long chunks, long long words) {
    const long long row_bytes = (k + 1) / 2;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (long long)gridDim.x * blockDim.x) {
        const int st = (int)(i & 3), lane = (int)(i >> 2) & 31;
        const long long tile = i >> 7, rt = tile / chunks, col = (tile % chunks) * 64 + (st >> 1) * 32 + (lane & 3) * 8 + (st & 1) * 4;
        unsigned word = 0;
        for (int half = 0; half < 2; ++half)
            for (int e = 0; e < 4; ++e) {
                const long long row = rt * 16 + (lane >> 2) + half * 8, cc = col + e;
                const unsigned v = row < n && cc < k ? (in[row * row_bytes + cc / 2] >> (4 * (cc & 1))) & 15u : 8u;
                word |= v << (4 * nibble(half, e));
            }
        codes[i] = word;
    }
}
template <typename U>
__global__ void q4_pack_scales_kernel(const U* __restrict__ in, U* __restrict__ out, long long n, long long groups, long long total) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long q = (i >> 4) % groups, row = (i >> 4) / groups * 16 + (i & 15);
        out[i] = row < n ? in[row * groups + q] : U(0);
    }
}

// The values that the codes stand for, row by row.  A thread has one word: four columns of two rows.
template <typename T>
__global__ void q4_dequantize_kernel(const uint32_t* __restrict__ codes, const void* __restrict__ scales, DType sdt, T* __restrict__ out, long long n,
                                     long long k, int group, long long chunks, long long groups, long long words) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (long long)gridDim.x * blockDim.x) {
        // neighbours write neighbouring columns
        const int c = (int)(i >> 1) & 3, st = (int)(i >> 3 & 1) * 2 + (int)(i & 1), g = (int)(i >> 4) & 7;
        const long long tile = i >> 7, rt = tile / chunks, col = (tile % chunks) * 64 + (i & 15) * 4;
        const unsigned w = codes[tile * 128 + (g * 4 + c) * 4 + st];
        if (col >= k) continue;
        const long long q = col / group;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const long long row = rt * 16 + g + half * 8;
            if (row >= n) continue;
            const float s = scale_at(scales, sdt, (rt * groups + q) * 16 + g + half * 8);
            Pack<T, 4> v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v.v[e] = from_f<T>((float)((int)((w >> (4 * nibble(half, e))) & 15u) - 8) * s);
            T* to = out + row * k + col;
            if (k % 4 == 0) *reinterpret_cast<Pack<T, 4>*>(to) = v;
            else
                for (int e = 0; e < 4 && col + e < k; ++e) to[e] = v.v[e];
        }
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// Rows of x as the product reads them: columns padded with zeros to whole chunks; a row of f32 as its three bf16 parts.
template <typename T>
__global__ void q4_stage_kernel(const T* __restrict__ x, long long rs, long long cs, uint16_t* __restrict__ out, long long rows, long long k, long long kp) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows * kp; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / kp, j = i - r * kp;
        const T v = j < k ? x[r * rs + j * cs] : from_f<T>(0.f);
        if constexpr (sizeof(T) == 4) {
            // towards zero, so that no part leaves the range; three parts of 8 bits hold all 24
            const __nv_bfloat16 a = __float2bfloat16_rz(v);
            const float r1 = isfinite(v) ? v - __bfloat162float(a) : 0.f;
            const __nv_bfloat16 b = __float2bfloat16_rz(r1), c = __float2bfloat16_rn(r1 - __bfloat162float(b));
            out[(r * 3) * kp + j] = __bfloat16_as_ushort(a);
            out[(r * 3 + 1) * kp + j] = __bfloat16_as_ushort(b);
            out[(r * 3 + 2) * kp + j] = __bfloat16_as_ushort(c);
        } else {
            out[i] = *reinterpret_cast<const uint16_t*>(&v);
        }
    }
}

struct Q4Params {
    const uint4* codes;
    const void* scales;
    const uint16_t* x;       // [columns][x_stride], 16-byte aligned rows, zeros to the end of the last chunk
    void* y;                 // [rows][n]
    long long x_stride, n;
    int columns, rows, parts;    // columns = rows * parts
    int chunks, groups, group_log2, row_tiles;
    DType scale_dtype;
    int chunks_per_cta;      // of the CTA's share of the columns
};

template <bool BF> __device__ __forceinline__ void expand(unsigned w, unsigned (&a)[4]) {
    if constexpr (BF) {
        // (code - 8) / 1024, exactly: x may be anywhere in the range of f32, and sums of 128 products must not leave it
        const __nv_bfloat162 unit = __halves2bfloat162(__ushort_as_bfloat16(0x3a80), __ushort_as_bfloat16(0x3a80));   // 2^-10
        const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0xbe08), __ushort_as_bfloat16(0xbe08));    // -136 * 2^-10
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), unit, off);
            a[i] = *reinterpret_cast<const unsigned*>(&d);
        }
    } else {
        // the high nibbles of each byte are 16 (code) above 1024: a sixteenth of that, less 72
        const __half2 off = __half2half2(__ushort_as_half(0x6408)), sixteenth = __half2half2(__ushort_as_half(0x2c00)), off16 = __half2half2(__ushort_as_half(0xd480));
        const unsigned u = w >> 8;
        const unsigned v[4] = {(w & 0x000f000fu) | 0x64006400u, (w & 0x00f000f0u) | 0x64006400u, (u & 0x000f000fu) | 0x64006400u, (u & 0x00f000f0u) | 0x64006400u};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 x = *reinterpret_cast<const __half2*>(&v[i]);
            const __half2 d = i & 1 ? __hfma2(x, sixteenth, off16) : __hsub2(x, off);
            a[i] = *reinterpret_cast<const unsigned*>(&d);
        }
    }
}
template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if constexpr (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One CTA: TILES row tiles and a share of the columns, which its warps divide chunk by chunk.  The CTAs of a cluster have the
// shares of the same rows; the first adds them up, in their order.
template <typename T, bool BF, bool G32, int CT, int TILES>
__global__ void __launch_bounds__(kWarps * 32) q4_rows_kernel(const __grid_constant__ Q4Params p) {
    constexpr int NB = 4;                                   // chunks whose words a warp has in flight
    constexpr int NS = G32 ? 2 : 1;                         // groups of a chunk that have scales of their own
    extern __shared__ __align__(16) float sums[];           // [warp][TILES * 16][CT * 8]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int shares = (int)cluster.num_blocks(), share = (int)cluster.block_rank();
    const int rt0 = (int)(blockIdx.x / shares) * TILES;
    const int k0 = share * p.chunks_per_cta, k1 = min(p.chunks, k0 + p.chunks_per_cta);

    float total[TILES][CT][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int n = 0; n < CT; ++n) total[t][n][0] = total[t][n][1] = total[t][n][2] = total[t][n][3] = 0.f;

    const uint4* w[TILES];
    long long sc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const long long rt = min(rt0 + t, p.row_tiles - 1);
        w[t] = p.codes + rt * p.chunks * 32 + lane;
        sc[t] = rt * p.groups * 16 + g;
    }
    const uint16_t* xr[CT];
    bool have[CT];
#pragma unroll
    for (int n = 0; n < CT; ++n) {
        have[n] = n * 8 + g < p.columns;
        xr[n] = p.x + (long long)min(n * 8 + g, p.columns - 1) * p.x_stride + c * 8;
    }
    for (int base = k0 + warp; base < k1; base += kWarps * NB) {
        uint4 words[NB][TILES];
        float scale[NB][TILES][NS][2];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int kc = min(base + i * kWarps, k1 - 1);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                words[i][t] = __ldcs(w[t] + (long long)kc * 32);
#pragma unroll
                for (int q = 0; q < NS; ++q) {
                    const long long at = sc[t] + (long long)min((kc * 64 + q * 32) >> p.group_log2, p.groups - 1) * 16;
                    scale[i][t][q][0] = scale_at(p.scales, p.scale_dtype, at);
                    scale[i][t][q][1] = scale_at(p.scales, p.scale_dtype, at + 8);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int kc = base + i * kWarps;
            if (kc < k1) {
                float acc[TILES][CT][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half == 0 || G32) {
#pragma unroll
                        for (int t = 0; t < TILES; ++t)
#pragma unroll
                            for (int n = 0; n < CT; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
                    }
                    uint4 x[CT];
#pragma unroll
                    for (int n = 0; n < CT; ++n)
                        x[n] = have[n] ? __ldg(reinterpret_cast<const uint4*>(xr[n] + (long long)kc * 64 + half * 32)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        unsigned a[4];
                        expand<BF>(half ? words[i][t].z : words[i][t].x, a);
#pragma unroll
                        for (int n = 0; n < CT; ++n) mma<BF>(acc[t][n], a, x[n].x, x[n].y);
                        expand<BF>(half ? words[i][t].w : words[i][t].y, a);
#pragma unroll
                        for (int n = 0; n < CT; ++n) mma<BF>(acc[t][n], a, x[n].z, x[n].w);
                    }
                    if (half == 1 || G32) {
#pragma unroll
                        for (int t = 0; t < TILES; ++t)
#pragma unroll
                            for (int n = 0; n < CT; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) total[t][n][e] += acc[t][n][e] * scale[i][t][G32 ? half : 0][e >> 1];
                    }
                }
            }
        }
    }

    constexpr int COLS = CT * 8, ROWS = TILES * 16;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int n = 0; n < CT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sums[(warp * ROWS + t * 16 + g + (e >> 1) * 8) * COLS + n * 8 + c * 2 + (e & 1)] = total[t][n][e];
    __syncthreads();
    // the first warp's place takes the CTA's sum; every value is added up by one thread
    for (int i = threadIdx.x; i < ROWS * COLS; i += kWarps * 32) {
        float s = sums[i];
#pragma unroll
        for (int v = 1; v < kWarps; ++v) s += sums[v * ROWS * COLS + i];
        sums[i] = s;
    }
    if (shares > 1) cluster.sync();
    else __syncthreads();
    if (share == 0) {
        for (int i = threadIdx.x; i < ROWS * p.rows; i += kWarps * 32) {
            const int r = i % ROWS, m = i / ROWS;
            const long long row = (long long)rt0 * 16 + r;
            if (row >= p.n) continue;
            float y = 0.f;
            for (int part = p.parts - 1; part >= 0; --part) {       // the smallest part of a row of f32 first
                const int at = r * COLS + m * p.parts + part;
                float s = sums[at];
                for (int v = 1; v < shares; ++v) s += cluster.map_shared_rank(sums, v)[at];
                y += s;
            }
            ((T*)p.y)[(long long)m * p.n + row] = from_f<T>(BF ? y * 1024.f : y);
        }
    }
    if (shares > 1) cluster.sync();                         // nobody leaves while its sums may be read
}

template <typename T, bool BF, bool G32, int CT, int TILES>
void launch_rows(Device& dev, const Q4Params& p, int shares) {
    auto kernel = q4_rows_kernel<T, BF, G32, CT, TILES>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.row_tiles + TILES - 1) / TILES * shares));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = sizeof(float) * kWarps * TILES * 16 * CT * 8;    // 32 KiB at most
    cfg.stream = dev.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)shares, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    dev.begin_launch("q4_rows");
    if (!dev.dry) WGF_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    dev.end_launch();
}
template <typename T, bool BF, bool G32>
void dispatch_rows(Device& dev, const Q4Params& p, int ct, int tiles, int shares) {
    if (ct == 1 && tiles == 1) launch_rows<T, BF, G32, 1, 1>(dev, p, shares);
    else if (ct == 1) launch_rows<T, BF, G32, 1, 2>(dev, p, shares);
    else if (ct == 2 && tiles == 1) launch_rows<T, BF, G32, 2, 1>(dev, p, shares);
    else if (ct == 2) launch_rows<T, BF, G32, 2, 2>(dev, p, shares);
    else if (tiles == 1) launch_rows<T, BF, G32, 4, 1>(dev, p, shares);
    else launch_rows<T, BF, G32, 4, 2>(dev, p, shares);
}
template <typename T, bool BF>
void dispatch_group(Device& dev, const Q4Params& p, int ct, int tiles, int shares) {
    if (p.group_log2 == 5) dispatch_rows<T, BF, true>(dev, p, ct, tiles, shares);
    else dispatch_rows<T, BF, false>(dev, p, ct, tiles, shares);
}

unsigned grid_for(Device& dev, long long items) { return (unsigned)std::min<long long>((items + 255) / 256, (long long)dev.sm_count * 32); }

Q4Ref make_q4(const DeviceRef& devref, int64_t n, int64_t k, int64_t group, DType scale_dtype) {
    WGF_CHECK(group == 32 || group == 64 || group == 128, WGF_ERR_INVALID_ARGUMENT, "4-bit weights take groups of 32, 64 or 128 columns");
    WGF_CHECK(n >= 1 && k >= 1, WGF_ERR_SHAPE, "4-bit weights must have at least one row and one column");
    WGF_CHECK(n < (1ll << 31) - 64 && k < (1ll << 30), WGF_ERR_UNSUPPORTED, "4-bit weights: extents too large");
    devref->refuse_while_recording("making 4-bit weights");
    auto w = std::make_shared<Q4Weight>();
    w->dev = devref;
    w->n = n;
    w->k = k;
    w->group = group;
    w->row_tiles = (n + 15) / 16;
    w->chunks = (k + 63) / 64;
    w->groups = (k + group - 1) / group;
    w->scale_dtype = scale_dtype;
    WGF_CHECK(w->row_tiles < (1ll << 46) / (w->chunks * 512), WGF_ERR_OOM, "the weights do not fit in memory");
    devref->make_current();
    w->codes = devref->alloc((size_t)(w->row_tiles * w->chunks) * 512, false);
    w->scales = devref->alloc((size_t)(w->row_tiles * w->groups) * 16 * dtype_size(scale_dtype), false);
    return w;
}

}  // namespace

Q4Ref q4_quantize(const DeviceRef& devref, const TensorData& x, int64_t group) {
    Device& dev = *devref;
    WGF_CHECK(x.layout.rank() == 2, WGF_ERR_RANK, "4-bit weights are made from a [rows, columns] tensor");
    Q4Ref w = make_q4(devref, x.layout.shape[0], x.layout.shape[1], group, x.dtype);
    dev.wait_for(*x.buf);
    // the groups of whole chunks: behind the last column there are codes (of zero), though no scales
    const long long padded = (w->chunks * 64 + group - 1) / group, jobs = w->row_tiles * padded * 8;
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        dev.begin_launch("q4_quantize");
        if (!dev.dry)
            q4_quantize_kernel<T><<<grid_for(dev, jobs * 32), 256, 0, dev.stream>>>((const T*)x.base_ptr(), x.layout.strides[0], x.layout.strides[1],
                (uint32_t*)w->codes->ptr, (T*)w->scales->ptr, w->n, w->k, (int)group, w->chunks, w->groups, padded, jobs);
        dev.end_launch();
    };
    if (x.dtype == DType::F32) go(0.f);
    else if (x.dtype == DType::F16) go(__half());
    else go(__nv_bfloat16());
    return w;
}

Q4Ref q4_from_host(const DeviceRef& devref, int64_t n, int64_t k, int64_t group, const uint8_t* codes, DType scale_dtype, const void* scales) {
    Device& dev = *devref;
    Q4Ref w = make_q4(devref, n, k, group, scale_dtype);
    const size_t cb = (size_t)n * ((k + 1) / 2), sb = (size_t)(n * w->groups) * dtype_size(scale_dtype);
    BufferRef c = dev.alloc(cb, false), s = dev.alloc(sb, false);
    dev.upload(*c, 0, codes, cb);
    dev.upload(*s, 0, scales, sb);
    const long long words = w->row_tiles * w->chunks * 128, total = w->row_tiles * w->groups * 16;
    dev.begin_launch("q4_pack");
    if (!dev.dry) q4_pack_kernel<<<grid_for(dev, words), 256, 0, dev.stream>>>((const uint8_t*)c->ptr, (uint32_t*)w->codes->ptr, n, k, w->chunks, words);
    dev.end_launch();
    dev.begin_launch("q4_pack");
    if (!dev.dry) {
        if (scale_dtype == DType::F32) q4_pack_scales_kernel<uint32_t><<<grid_for(dev, total), 256, 0, dev.stream>>>((const uint32_t*)s->ptr, (uint32_t*)w->scales->ptr, n, w->groups, total);
        else q4_pack_scales_kernel<uint16_t><<<grid_for(dev, total), 256, 0, dev.stream>>>((const uint16_t*)s->ptr, (uint16_t*)w->scales->ptr, n, w->groups, total);
    }
    dev.end_launch();
    return w;
}

TensorData q4_dequantize(Device& dev, const Q4Weight& w, DType dtype) {
    dev.make_current();
    dev.note_recorded_buffer(w.codes);
    dev.note_recorded_buffer(w.scales);
    TensorData out;
    out.dtype = dtype;
    out.layout = Layout::contiguous({w.n, w.k});
    out.buf = dev.alloc((size_t)(w.n * w.k) * dtype_size(dtype), false);
    const long long words = w.row_tiles * w.chunks * 128;
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        dev.begin_launch("q4_dequantize");
        if (!dev.dry)
            q4_dequantize_kernel<T><<<grid_for(dev, words), 256, 0, dev.stream>>>((const uint32_t*)w.codes->ptr, w.scales->ptr, w.scale_dtype,
                (T*)out.buf->ptr, w.n, w.k, (int)w.group, w.chunks, w.groups, words);
        dev.end_launch();
    };
    if (dtype == DType::F32) go(0.f);
    else if (dtype == DType::F16) go(__half());
    else go(__nv_bfloat16());
    return out;
}

TensorData run_matmul_q4(Device& dev, const TensorData& x_in, const Q4Weight& w) {
    dev.make_current();
    const int r = x_in.layout.rank();
    TensorData x = x_in, out;
    // leading axes as one: a matrix of rows
    if (r > 2 && !(x.layout.is_dense() && !x.layout.allocation_overlaps())) x = run_compact(dev, x);
    const int64_t rows = x_in.layout.numel() / w.k;
    x.layout.shape = {rows, w.k};
    x.layout.strides = {r == 2 ? x.layout.strides[0] : w.k, x.layout.strides[r - 1]};
    std::vector<int64_t> shape = x_in.layout.shape;
    shape[r - 1] = w.n;
    out.dtype = x.dtype;
    out.layout = Layout::contiguous(shape);
    if (rows == 0) {
        out.buf = dev.alloc(1, false);
        return out;
    }
    dev.wait_for(*x.buf);
    const int parts = x.dtype == DType::F32 ? 3 : 1;
    if (rows * parts > 32) {
        TensorData full = q4_dequantize(dev, w, x.dtype);
        full.layout.shape = {w.k, w.n};
        full.layout.strides = {1, w.k};
        TensorData y = run_matmul(dev, x, full);
        y.layout = out.layout;
        return y;
    }
    dev.note_recorded_buffer(w.codes);
    dev.note_recorded_buffer(w.scales);
    out.buf = dev.alloc((size_t)(rows * w.n) * dtype_size(x.dtype), false);
    Q4Params p{};
    p.codes = (const uint4*)w.codes->ptr;
    p.scales = w.scales->ptr;
    p.y = out.buf->ptr;
    p.n = w.n;
    p.rows = (int)rows;
    p.parts = parts;
    p.columns = (int)rows * parts;
    p.chunks = (int)w.chunks;
    p.groups = (int)w.groups;
    p.group_log2 = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    p.row_tiles = (int)w.row_tiles;
    p.scale_dtype = w.scale_dtype;
    BufferRef staged;
    if (parts == 1 && w.k % 64 == 0 && x.layout.strides[1] == 1 && (rows == 1 || x.layout.strides[0] % 8 == 0) && (uintptr_t)x.base_ptr() % 16 == 0) {
        p.x = (const uint16_t*)x.base_ptr();
        p.x_stride = x.layout.strides[0];
    } else {
        const long long kp = w.chunks * 64;
        staged = dev.alloc((size_t)(p.columns * kp) * 2, false);
        p.x = (const uint16_t*)staged->ptr;
        p.x_stride = kp;
        dev.begin_launch("q4_stage");
        if (!dev.dry) {
            const unsigned grid = grid_for(dev, rows * kp);
            if (x.dtype == DType::F32) q4_stage_kernel<float><<<grid, 256, 0, dev.stream>>>((const float*)x.base_ptr(), x.layout.strides[0], x.layout.strides[1], (uint16_t*)staged->ptr, rows, w.k, kp);
            else q4_stage_kernel<__half><<<grid, 256, 0, dev.stream>>>((const __half*)x.base_ptr(), x.layout.strides[0], x.layout.strides[1], (uint16_t*)staged->ptr, rows, w.k, kp);
        }
        dev.end_launch();
    }
    const int ct = p.columns <= 8 ? 1 : p.columns <= 16 ? 2 : 4;
    const int tiles = 1;
    // CTAs for the whole GPU, as long as each warp has a chunk
    int shares = 1;
    while (shares < 8 && (w.row_tiles / tiles) * shares < 2 * dev.sm_count && w.chunks / (shares * 2) >= kWarps) shares *= 2;
    p.chunks_per_cta = (int)((w.chunks + shares - 1) / shares);
    if (x.dtype == DType::F16) dispatch_group<__half, false>(dev, p, ct, tiles, shares);
    else if (x.dtype == DType::BF16) dispatch_group<__nv_bfloat16, true>(dev, p, ct, tiles, shares);
    else dispatch_group<float, true>(dev, p, ct, tiles, shares);
    return out;
}

}  // namespace wgf
