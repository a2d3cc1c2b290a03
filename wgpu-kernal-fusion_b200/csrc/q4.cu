// Products with 4-bit weights.
//
//   y[m, n] = sum over groups of columns of scale[n, group] * sum_{k in group} x[m, k] * (code[n, k] - 8)
//
// The weights are stored in tiles of 16 rows by 64 columns, 512 bytes, in the order in which the lanes of a warp want them
// as the A operand of four m16n8k16 instructions: lane (g, c) has 16 bytes, one word a step, with columns
// 32 (step / 2) + 8 c + 4 (step % 2) .. + 3 of rows g and g + 8, so that two steps are 32 columns in a row.  Within a
// word the two values that become one register are 16 bits apart:
//   nibble  0 / 4: row g, columns 0 / 1      1 / 5: row g + 8, columns 0 / 1
//           2 / 6: row g, columns 2 / 3      3 / 7: row g + 8, columns 2 / 3
// The scales of a tile's 16 rows stand together for each group, those of rows g and g + 8 side by side.
//
// Few rows of x: every weight is read once, half a byte each, and used for at most a few multiplications, so memory is the
// bound, and next to it the instructions that turn words into operands (about 80 of f16 and 85 of bf16 for the 16 x 64 weights of a
// unit; 11008 x 4096 weights are 74 units for each scheduler of the GPU).  The instruction's eight columns are the
// rows of x; codes become f16 or bf16 exactly, and sums are f32 within a group and across groups.  A row of f32 takes
// three columns: its bf16 parts, which together have its 24 bits.  The product does not go through tensor memory: the
// converted codes would have to be written there, or to shared memory, first, and for eight columns the conversion, not the product, is the work.
// One row through 11008 x 4096, groups of 128, f16, recorded: 10.7 to 12.3 us a pass (such passes come in steps of 2.05), 10.5 in a row of
// products (23 MB; 3.5 at the measured rate of memory); 16.5 with a CTA for each row tile, whose first loads, staging of x and sums were not
// overlapped with anything, and 22 where a scale was converted, and so waited for, in the turn that called for it.
// Seven rows of bf16 through 4096 x 11008: 14.7 us a pass, 13 in a row of products.
// More rows: in blocks, along the grid's second axis, or on the tensor cores (q4_tc.cu; choose_way has the times).
#include <algorithm>

#include <cooperative_groups.h>

#include "decode.hpp"
#include "decode_common.cuh"
#include "q4_tc.hpp"

namespace wgf {

using namespace decode;
namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 16;        // of a CTA of the product; one CTA a SM
constexpr int kMaxTiles = 32;     // row tiles of a CTA
constexpr int kSmem = 227 * 1024;
// A unit, 16 rows by 64 columns, in a warp's ring: its words, and the scales of every lane's two rows
__host__ __device__ constexpr int ring_unit(bool wide, bool g32) { return 512 + 32 * (wide ? 8 : 4) * (g32 ? 2 : 1); }

// Where the scale of a tile's row is among the 16 of a group
__host__ __device__ __forceinline__ int scale_slot(int row) { return (row & 7) * 2 + (row >> 3); }

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
            if (lane == 0 && q < groups) scales[(rt * groups + q) * 16 + scale_slot(g + half * 8)] = st;
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
        out[i - (i & 15) + scale_slot((int)(i & 15))] = row < n ? in[row * groups + q] : U(0);
    }
}

// The values that the codes stand for, row by row, zeros between the last column and the end of a padded row.  A warp has tiles
// of kSpan chunks in a row, a lane eight columns of rows g and g + 8 at a time.  11008 x 4096 as f16: 28 us; with a thread for each
// word, whose place took four divisions of 64 bits, 52.
constexpr int kSpan = 4;
template <typename T>
__global__ void q4_dequantize_kernel(const uint4* __restrict__ codes, const void* __restrict__ scales, DType sdt, T* __restrict__ out, long long n,
                                     long long k, long long stride, int group_log2, long long chunks, long long groups, long long spans, long long jobs) {
    typedef Pack<T, 16 / (int)sizeof(T)> V;
    constexpr int PER = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const bool wide = stride % PER == 0;
    for (long long job = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); job < jobs; job += (long long)gridDim.x * (blockDim.x >> 5)) {
        const long long rt = job / spans, first = (job - rt * spans) * kSpan, row = rt * 16 + g;
#pragma unroll
        for (int i = 0; i < kSpan; ++i) {
            const long long chunk = first + i;
            if (chunk >= chunks) break;
            const uint4 w = codes[(rt * chunks + chunk) * 32 + lane];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const long long col = chunk * 64 + half * 32 + c * 8;
                if (col >= stride) continue;
                const unsigned word[2] = {half ? w.z : w.x, half ? w.w : w.y};
                const long long q = min(col >> group_log2, groups - 1);
#pragma unroll
                for (int low = 0; low < 2; ++low) {
                    if (row + low * 8 >= n) continue;
                    const float s = scale_at(scales, sdt, (rt * groups + q) * 16 + g * 2 + low);
                    T v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = from_f<T>((float)((int)((word[e >> 2] >> (4 * nibble(low, e & 3))) & 15u) - 8) * s);
                    if (col + 8 > k)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e >= k) v[e] = from_f<T>(0.f);
                    T* to = out + (row + low * 8) * stride + col;
                    if (wide && col + 8 <= stride) {
#pragma unroll
                        for (int e = 0; e < 8; e += PER) {
                            V p;
#pragma unroll
                            for (int f = 0; f < PER; ++f) p.v[f] = v[e + f];
                            *reinterpret_cast<V*>(to + e) = p;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e < stride) to[e] = v[e];
                    }
                }
            }
        }
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
struct Q4Params {
    const uint4* codes;
    const void* scales;
    const void* x;           // [rows][k], last axis dense
    void* y;                 // [rows][n]
    long long x_stride, n, k;
    int rows, columns;       // of a block of rows; columns of the instruction: one for each row, three for one of f32
    int all_rows;            // blocks of rows lie along the grid's second axis
    int chunks, groups, group_log2, row_tiles;
    DType scale_dtype;
    int tiles, share_chunks; // row tiles of a cluster, chunks of a CTA's share of them
    int aligned;             // 16-bit rows of x in 16-byte pieces
};

// Eight values of a row of x from column `at` on, as one 16-byte operand for each part; zeros behind the end of the row.
template <typename T> __device__ __forceinline__ void operands(const T* row, long long at, long long k, uint4 (&out)[sizeof(T) == 4 ? 3 : 1]) {
    T x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = at + e < k ? row[at + e] : from_f<T>(0.f);
    unsigned short h[sizeof(T) == 4 ? 3 : 1][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 4) {
            // the bf16 parts of x: cut towards zero, so that none leaves the range; three of 8 bits hold all 24
            const __nv_bfloat16 p0 = __float2bfloat16_rz(x[e]);
            const float r1 = isfinite(x[e]) ? x[e] - __bfloat162float(p0) : 0.f;
            const __nv_bfloat16 p1 = __float2bfloat16_rz(r1), p2 = __float2bfloat16_rn(r1 - __bfloat162float(p1));
            h[0][e] = __bfloat16_as_ushort(p0);
            h[1][e] = __bfloat16_as_ushort(p1);
            h[2][e] = __bfloat16_as_ushort(p2);
        } else {
            h[0][e] = *reinterpret_cast<const unsigned short*>(&x[e]);
        }
    }
#pragma unroll
    for (int q = 0; q < (sizeof(T) == 4 ? 3 : 1); ++q)
        out[q] = make_uint4(h[q][0] | (unsigned)h[q][1] << 16, h[q][2] | (unsigned)h[q][3] << 16, h[q][4] | (unsigned)h[q][5] << 16, h[q][6] | (unsigned)h[q][7] << 16);
}

// Rows of f32 as their parts, for the tensor cores: [rows / 32][part][32][stride]
__global__ void q4_split_kernel(const float* __restrict__ x, long long x_stride, long long rows, long long k, __nv_bfloat16* __restrict__ out, long long stride) {
    const long long pieces = stride / 8, total = rows * pieces;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / pieces, at = (i - row * pieces) * 8;
        uint4 part[3];
        operands<float>(x + row * x_stride, at, k, part);
        __nv_bfloat16* to = out + (row / kSplitRows * 3 * kSplitRows + row % kSplitRows) * stride + at;
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(to + q * kSplitRows * stride) = part[q];
    }
}

// The scales of rows g and g + 8, from what a lane's copy brought
template <bool WIDE> __device__ __forceinline__ float2 two_scales(unsigned at, bool half) {
    if constexpr (WIDE) return shared_float2(at);
    const unsigned v = shared_word(at);
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return make_float2(half ? h.x : __uint_as_float(v << 16), half ? h.y : __uint_as_float(v & 0xffff0000u));
}

// A word's codes less 8 as the operand of one instruction, exactly.
// bf16: (code - 8) / 1024.  x may be anywhere in the range of f32, and sums of 128 products must not leave it.
// f16: the nibbles of rows g under the exponent of 1024, less 1032; those of rows g + 8 stand four bits higher, so there it is a
// sixteenth of 1024 + 16 code, less 72, as one fused multiply-add.
template <bool BF> __device__ __forceinline__ void expand(unsigned w, unsigned (&a)[4]) {
    if constexpr (BF) {
        const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0xbe08), __ushort_as_bfloat16(0xbe08));    // -136 / 1024
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned v = ((w >> (4 * i)) & 0x000f000fu) | 0x3e003e00u;      // (128 + code) / 1024
            const __nv_bfloat162 d = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
            a[i] = *reinterpret_cast<const unsigned*>(&d);
        }
    } else {
        const __half2 off = __half2half2(__ushort_as_half(0xe408)), sixteenth = __half2half2(__ushort_as_half(0x2c00)), low = __half2half2(__ushort_as_half(0xd480));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const unsigned u = i ? w >> 8 : w, x = (u & 0x000f000fu) | 0x64006400u, y = (u & 0x00f000f0u) | 0x64006400u;
            const __half2 d = __hadd2(*reinterpret_cast<const __half2*>(&x), off), e = __hfma2(*reinterpret_cast<const __half2*>(&y), sixteenth, low);
            a[i] = *reinterpret_cast<const unsigned*>(&d);
            a[i + 1] = *reinterpret_cast<const unsigned*>(&e);
        }
    }
}
template <bool BF> __device__ __forceinline__ float operand_unit() { return BF ? 1024.f : 1.f; }

template <bool BF> __device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, bool fresh) {
    // fresh: the accumulator starts from zero
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fresh ? 0.f : d[i];
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// One CTA has some row tiles and a share of the columns; their (tile, chunk) units in a row are cut into equal stretches for
// its warps.  A warp has the words and scales of DEPTH units on their way into a ring of its own in shared memory, each
// lane what it will read itself, the first of them while x is brought there (512 bytes for half a chunk of eight columns, in
// the order in which lanes read them).  It puts its sums down where a tile or its stretch ends.  The CTAs of a cluster have
// the shares of the same rows.  Sums are added up in the order of the warps and of the CTAs.
template <typename T, bool WIDE, bool G32, int CT, int DEPTH>
__global__ void __launch_bounds__(kWarps * 32, 1) q4_rows_kernel(const __grid_constant__ Q4Params p) {
    constexpr bool BF = !std::is_same<T, __half>::value;
    constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
    constexpr int NS = G32 ? 2 : 1;                         // groups of a chunk that have scales of their own
    // The halves of a chunk have sums of their own where their scales differ, and for bf16, whose products then do not wait for one another (one
    // row through 11008 x 4096 11.1 us, 11.2 with one sum); f16 and f32 are faster with fewer instructions (10.5 instead of 10.8; 9.3 instead of 9.5).
    constexpr bool APART = G32 || std::is_same<T, __nv_bfloat16>::value;
    constexpr int COLS = CT * 8, SLOT = 16 * COLS;
    constexpr int UNIT = ring_unit(WIDE, G32), SB = WIDE ? 8 : 4;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char* ring = smem + (threadIdx.x >> 5) * (DEPTH * UNIT);   // [unit]{ 512 bytes of words; the lanes' scales }
    uint4* xs = reinterpret_cast<uint4*>(smem + kWarps * DEPTH * UNIT); // [chunk][half][column][4], and 16 bytes of zeros
    float* sums = reinterpret_cast<float*>(xs + p.share_chunks * p.columns * 8 + 1);     // [slot][row][column]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int shares = (int)cluster.num_blocks(), share = (int)cluster.block_rank();
    const int rt0 = (int)(blockIdx.x / shares) * p.tiles, tiles = min(p.tiles, p.row_tiles - rt0);
    const int k0 = share * p.share_chunks, nk = min(p.chunks - k0, p.share_chunks);
    const T* x_rows = (const T*)p.x + (long long)blockIdx.y * p.rows * p.x_stride;
    const int rows = min(p.rows, p.all_rows - (int)blockIdx.y * p.rows);
    const int units = tiles * nk, each = (units + kWarps - 1) / kWarps;
    const int u0 = min(units, warp * each), mine = min(units, u0 + each) - u0;

    // pieces of rows of x, eight values each: copied as they are where they can be
    const bool copied = sizeof(T) == 2 && p.aligned;
    if (copied) {
        for (int m = 0; m < rows; ++m) {
            const T* row = x_rows + (long long)m * p.x_stride + (long long)k0 * 64;
            for (int q = threadIdx.x; q < nk * 8; q += kWarps * 32) {
                uint4* to = xs + ((q >> 2) * p.columns + m) * 4 + (q & 3);
                if ((long long)k0 * 64 + q * 8 < p.k) copy16(to, row + q * 8);
                else *to = make_uint4(0, 0, 0, 0);
            }
        }
    }
    copies_commit();

    // The unit that is called for next, as offsets from the CTA's first: 16-byte pieces of codes, pairs of scales
    int tile = u0 / nk, at = u0 - tile * nk, next = k0 + at;
    const uint4* codes = p.codes + ((long long)rt0 * p.chunks) * 32;
    const unsigned char* scales = (const unsigned char*)p.scales + (long long)rt0 * p.groups * 8 * SB;
    unsigned w = (unsigned)(tile * p.chunks + next) * 32 + lane, sc = (unsigned)(tile * p.groups) * 8 + g;
    const unsigned over = (p.chunks - nk) * 32;             // from the end of a share to the next tile's
    int left = k0 + nk - next;                              // units of this tile that are still to be called for
    const int group_shift = p.group_log2 - 6;
    auto bring = [&](unsigned slot) {
        copy16_at(slot + lane * 16, codes + w);
        if constexpr (G32) {
            copy_at<SB>(slot + 512 + lane * SB, scales + (size_t)(sc + next * 16) * SB);
            copy_at<SB>(slot + 512 + (32 + lane) * SB, scales + (size_t)(sc + min(next * 2 + 1, p.groups - 1) * 8) * SB);
        } else {
            copy_at<SB>(slot + 512 + lane * SB, scales + (size_t)(sc + (next >> group_shift) * 8) * SB);
        }
        w += 32;
        ++next;
        if (--left == 0) {
            left = nk;
            next = k0;
            w += over;
            sc += p.groups * 8;
        }
    };
    const unsigned ring0 = shared_address(ring);
#pragma unroll 4
    for (int i = 0; i < DEPTH; ++i) {
        if (i < mine) bring(ring0 + i * UNIT);
        copies_commit();
    }

    if (threadIdx.x == 0) xs[nk * 8 * p.columns] = make_uint4(0, 0, 0, 0);
    if (copied) {
        copies_wait<DEPTH>();
    } else {
        for (int m = 0; m < rows; ++m)
#pragma unroll 2
            for (int q = threadIdx.x; q < nk * 8; q += kWarps * 32) {
                uint4 v[PARTS];
                operands<T>(x_rows + (long long)m * p.x_stride, (long long)k0 * 64 + q * 8, p.k, v);
#pragma unroll
                for (int e = 0; e < PARTS; ++e) xs[((q >> 2) * p.columns + m * PARTS + e) * 4 + (q & 3)] = v[e];
            }
    }
    __syncthreads();

    float total[CT][4];
#pragma unroll
    for (int n = 0; n < CT; ++n) total[n][0] = total[n][1] = total[n][2] = total[n][3] = 0.f;
    // a lane whose column of the instruction is not in use reads the zeros behind x, over and over
    unsigned x0[CT], x_step[CT];
#pragma unroll
    for (int n = 0; n < CT; ++n) {
        const bool have = n * 8 + g < rows * PARTS;
        x0[n] = shared_address(have ? xs + n * 32 + lane : xs + nk * 8 * p.columns);
        x_step[n] = have ? p.columns * 128 : 0;
    }
    const bool half_scales = p.scale_dtype == DType::F16;
    float* put = sums + (tile + warp) * SLOT + g * COLS + c * 2;       // every (tile, warp) that meet have a slot of their own
    auto put_down = [&] {
        const float unit = operand_unit<BF>();
#pragma unroll
        for (int n = 0; n < CT; ++n) {
            *reinterpret_cast<float2*>(put + n * 8) = make_float2(total[n][0] * unit, total[n][1] * unit);
            *reinterpret_cast<float2*>(put + 8 * COLS + n * 8) = make_float2(total[n][2] * unit, total[n][3] * unit);
            total[n][0] = total[n][1] = total[n][2] = total[n][3] = 0.f;
        }
        put += SLOT;
    };
    const unsigned ring_end = ring0 + DEPTH * UNIT;
    unsigned slot = ring0 + lane * 16;
    int ahead = mine - DEPTH;                               // units still to be called for
    for (int done = 0; done < mine;) {
        // a tile's units
        const int stretch = min(nk - at, mine - done);
        done += stretch;
        unsigned xl[CT];
#pragma unroll
        for (int n = 0; n < CT; ++n) xl[n] = x0[n] + at * x_step[n];
        at = 0;
#pragma unroll 2
        for (int i = 0; i < stretch; ++i) {
            copies_wait<DEPTH - 1>();
            const uint4 words = shared_16(slot);
            float2 s[NS];
#pragma unroll
            for (int q = 0; q < NS; ++q) s[q] = two_scales<WIDE>(slot - lane * (16 - SB) + 512 + q * 32 * SB, half_scales);
            float acc[2][CT][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint4 x[CT];
#pragma unroll
                for (int n = 0; n < CT; ++n) x[n] = shared_16(xl[n] + (half ? x_step[n] / 2 : 0));
                unsigned a[4];
                expand<BF>(half ? words.z : words.x, a);
#pragma unroll
                for (int n = 0; n < CT; ++n) mma<BF>(acc[APART ? half : 0][n], a, x[n].x, x[n].y, half == 0 || APART);
                expand<BF>(half ? words.w : words.y, a);
#pragma unroll
                for (int n = 0; n < CT; ++n) mma<BF>(acc[APART ? half : 0][n], a, x[n].z, x[n].w, false);
            }
            if (ahead > 0) bring(slot - lane * 16);
            --ahead;
            copies_commit();
            slot += UNIT;
            if (slot >= ring_end) slot -= DEPTH * UNIT;
#pragma unroll
            for (int n = 0; n < CT; ++n) xl[n] += x_step[n];
#pragma unroll
            for (int n = 0; n < CT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (G32) total[n][e] += acc[0][n][e] * (e < 2 ? s[0].x : s[0].y) + acc[1][n][e] * (e < 2 ? s[1].x : s[1].y);
                    else total[n][e] += (APART ? acc[0][n][e] + acc[1][n][e] : acc[0][n][e]) * (e < 2 ? s[0].x : s[0].y);
                }
        }
        put_down();
    }
    __syncthreads();

    // What the CTA's warps have of a value, in their order
    auto warps_sum = [&](int t, int r, int column) {
        const int w0 = t * nk / each, w1 = ((t + 1) * nk - 1) / each;
        float s = 0.f;
        for (int v = w0; v <= w1; ++v) s += sums[((t + v) * 16 + r) * COLS + column];
        return s;
    };
    float* joint = sums + (p.tiles + kWarps) * SLOT;        // [tile][row][column]: this CTA's share
    if (shares > 1) {
        for (int i = threadIdx.x; i < tiles * 16 * p.columns; i += kWarps * 32) {
            const int column = i % p.columns, row = i / p.columns;
            joint[row * COLS + column] = warps_sum(row >> 4, row & 15, column);
        }
        cluster.sync();
    }
    // with shares, each CTA of the cluster adds up a part of the values
    for (int i = threadIdx.x + share * (kWarps * 32); i < tiles * 16 * rows; i += kWarps * 32 * shares) {
        const int r = i % (tiles * 16), m = i / (tiles * 16);
        const long long row = (long long)rt0 * 16 + r;
        if (row >= p.n) continue;
        float y = 0.f;
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q) {              // the smallest part of a row of f32 first
            const int column = m * PARTS + q;
            float s = 0.f;
            if (shares > 1) {
#pragma unroll 2
                for (int v = 0; v < shares; ++v) s += cluster.map_shared_rank(joint, v)[r * COLS + column];
            } else {
                s = warps_sum(r >> 4, r & 15, column);
            }
            y += s;
        }
        ((T*)p.y)[((long long)blockIdx.y * p.rows + m) * p.n + row] = from_f<T>(y);
    }
    if (shares > 1) cluster.sync();                         // nobody leaves while its sums may be read
}

// Shared memory of a CTA whose warps have `depth` units on their way
size_t rows_smem(int share_chunks, int columns, int tiles, int ct, int shares, int unit, int depth) {
    return (size_t)kWarps * depth * unit + (size_t)share_chunks * (columns * 128) + 16 +
           (size_t)(tiles + kWarps + (shares > 1 ? tiles : 0)) * 16 * ct * 8 * sizeof(float);
}

template <typename T, bool WIDE, bool G32, int CT, int DEPTH>
void launch_depth(Device& dev, const Q4Params& p, int shares) {
    auto kernel = q4_rows_kernel<T, WIDE, G32, CT, DEPTH>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.row_tiles + p.tiles - 1) / p.tiles * shares), (unsigned)((p.all_rows + p.rows - 1) / p.rows));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = rows_smem(p.share_chunks, p.columns, p.tiles, CT, shares, ring_unit(WIDE, G32), DEPTH);
    cfg.stream = dev.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)shares, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = shares > 1 ? 1 : 0;
    if (!dev.dry) {
        static unsigned long long done = 0;    // one bit a device; setting it twice does no harm
        if (dev.ordinal >= 64 || !(done >> dev.ordinal & 1)) {
            WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
            if (dev.ordinal < 64) done |= 1ull << dev.ordinal;
        }
    }
    dev.begin_launch("q4_rows");
    if (!dev.dry) WGF_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    dev.end_launch();
}
// As many units on their way as there is room for
template <typename T, bool WIDE, bool G32, int CT>
void launch_rows(Device& dev, const Q4Params& p, int shares) {
    const int most = (p.tiles * p.share_chunks + kWarps - 1) / kWarps;      // units of a warp
    if (CT == 1 && most > 8 && rows_smem(p.share_chunks, p.columns, p.tiles, CT, shares, ring_unit(WIDE, G32), 16) <= (size_t)kSmem)
        launch_depth<T, WIDE, G32, CT, CT == 1 ? 16 : 8>(dev, p, shares);
    else launch_depth<T, WIDE, G32, CT, 8>(dev, p, shares);
}
template <typename T>
void dispatch_rows(Device& dev, const Q4Params& p, int ct, int shares) {
    auto with = [&](auto wide, auto g32) {
        constexpr bool WIDE = decltype(wide)::value, G32 = decltype(g32)::value;
        if (ct == 1) launch_rows<T, WIDE, G32, 1>(dev, p, shares);
        else launch_rows<T, WIDE, G32, 2>(dev, p, shares);
    };
    const bool wide = p.scale_dtype == DType::F32;
    if (wide && p.group_log2 == 5) with(std::true_type(), std::true_type());
    else if (wide) with(std::true_type(), std::false_type());
    else if (p.group_log2 == 5) with(std::false_type(), std::true_type());
    else with(std::false_type(), std::false_type());
}

// How many clusters of 1, 2, 4 and 8 CTAs the GPU runs at once with one CTA a SM: fewer than its SMs would make, as a
// cluster's SMs have to be neighbours.
const int* clusters_at_once(Device& dev) {
    static int known[64][4];
    int* k = known[dev.dry || dev.ordinal >= 64 ? 63 : dev.ordinal];
    if (k[0]) return k;
    k[1] = k[2] = k[3] = 0;
    for (int i = 1; i < 4; ++i) {
        k[i] = dev.sm_count >> i;
        if (dev.dry) continue;
        auto kernel = q4_rows_kernel<__half, false, false, 1, 8>;
        WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(dev.sm_count << i));
        cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = kSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {1u << i, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        k[i] = std::max(std::min(n, k[i]), 1);
    }
    k[0] = dev.sm_count;
    return k;
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

static int group_log2(const Q4Weight& w) { return w.group == 32 ? 5 : w.group == 64 ? 6 : 7; }

// [n, k] in rows of `stride` elements, zeros behind the last column
static TensorData dequantize_rows(Device& dev, const Q4Weight& w, DType dtype, int64_t stride) {
    dev.make_current();
    dev.note_recorded_buffer(w.codes);
    dev.note_recorded_buffer(w.scales);
    TensorData out;
    out.dtype = dtype;
    out.layout = Layout::contiguous({w.n, stride});
    out.buf = dev.alloc((size_t)(w.n * stride) * dtype_size(dtype), false);
    const long long spans = (w.chunks + kSpan - 1) / kSpan, jobs = w.row_tiles * spans;
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        dev.begin_launch("q4_dequantize");
        if (!dev.dry)
            q4_dequantize_kernel<T><<<grid_for(dev, jobs * 32), 256, 0, dev.stream>>>((const uint4*)w.codes->ptr, w.scales->ptr, w.scale_dtype,
                (T*)out.buf->ptr, w.n, w.k, stride, group_log2(w), w.chunks, w.groups, spans, jobs);
        dev.end_launch();
    };
    if (dtype == DType::F32) go(0.f);
    else if (dtype == DType::F16) go(__half());
    else go(__nv_bfloat16());
    return out;
}

TensorData q4_dequantize(Device& dev, const Q4Weight& w, DType dtype) { return dequantize_rows(dev, w, dtype, w.k); }

// How the product with few rows is dealt out: rows in blocks, row tiles of the weights to the SMs, or with shares of the
// columns to clusters of them.  x has to fit beside the sums.
struct RowsPlan {
    int shares = 0, tiles = 0, ct = 0, block_rows = 0;     // shares == 0: it does not fit
    double cost = 1e30;                                    // in the time that a SM takes for a unit with eight columns, about 21 ns
};
static RowsPlan plan_rows(Device& dev, const Q4Weight& w, int64_t rows, int parts) {
    RowsPlan best;
    const int* at_once = clusters_at_once(dev);
    const int unit = ring_unit(w.scale_dtype == DType::F32, w.group == 32);
    // Joining a cluster's sums costs more than it saves from clusters of four on (eight rows of f16 through 11008 x 4096: 21 us
    // with four, 13 with one), so those are for rows of x that fit in no other way.
    for (int s = 1, i = 0; i < 4 && (i < 2 || !best.shares); s *= 2, ++i)
        for (int ct : {1, 2}) {
            const int64_t most = ct * 8 / parts, blocks = (rows + most - 1) / most, block_rows = (rows + blocks - 1) / blocks, columns = block_rows * parts;
            if (blocks > 65535 || (ct == 2 && columns <= 8)) continue;
            const int64_t chunks = (w.chunks + s - 1) / s, clusters = at_once[i];
            const int64_t room = (int64_t)kSmem - (int64_t)rows_smem((int)std::min<int64_t>(chunks, 1 << 20), (int)columns, 0, ct, s, unit, 8);
            const int64_t fit = room / ((s > 1 ? 2 : 1) * 16 * ct * 8 * (int64_t)sizeof(float));      // tiles whose sums there is room for
            if ((s - 1) * chunks >= w.chunks || fit < 1) continue;
            const int64_t t = std::min<int64_t>({(w.row_tiles * blocks + clusters - 1) / clusters, w.row_tiles, fit, kMaxTiles});
            const int64_t turns = ((w.row_tiles + t - 1) / t * blocks + clusters - 1) / clusters;
            // the units, the bringing of x, what a CTA costs at its ends; and the joining
            const double cost = (double)turns * ((double)chunks * (t * (ct == 1 ? 1.0 : 1.4) + 0.13 * columns) + 40) + (s > 1 ? 40 + 0.8 * t * columns : 0);
            if (cost < best.cost) best = {s, (int)t, ct, (int)block_rows, cost};
        }
    return best;
}

// Which way rows take: in blocks through the kernel above, or through the tensor cores (q4_tc.cu).  Codes and scales enter both exactly, so that they differ
// in the order of f32 sums alone.  What each would take is estimated, in us.  Measured, blocks / tensor cores, f16 rows: 11008 x 4096, 32 rows 26 / 38,
// 48 rows 53 / 38, 500 rows 369 / 62; 4096 x 4096, 32 rows 14 / 16, 48 rows 18 / 17, 500 rows 149 / 32; 600 x 4000 in groups of 32, 100 rows 11 / 17, 500 rows
// 38 / 25; 1024 x 1024, 200 rows 10 / 11, 500 rows 24 / 13.  f32 rows, with the taking apart: 11008 x 4096, 6 rows 24 / 39, 12 rows 62 / 39;
// 4096 x 4096, 12 rows 18 / 18, 24 rows 52 / 18; 1024 x 1024, 48 rows 9 / 12, 100 rows 18 / 12.
enum class Q4Way { BLOCKS, TENSOR };
static Q4Way choose_way(const RowsPlan& plan, const Q4TcPlan& tc, int parts) {
    const double blocks = plan.shares ? 3.0 + 0.021 * plan.cost : 1e30;
    return blocks <= tc.us + (parts > 1 ? 2.0 : 0.0) ? Q4Way::BLOCKS : Q4Way::TENSOR;      // 2: taking x apart
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
    const RowsPlan plan = plan_rows(dev, w, rows, parts);
    // (rows that one block holds are read off the codes once: nothing is faster)
    const Q4TcPlan tc = rows > 8 || !plan.shares ? q4_tc_plan(dev, w, rows, parts) : Q4TcPlan();
    dev.note_recorded_buffer(w.codes);
    dev.note_recorded_buffer(w.scales);
    if (choose_way(plan, tc, parts) == Q4Way::TENSOR) {
        if (x.layout.strides[1] != 1 && w.k > 1) x = run_compact(dev, x);
        const int64_t kp = (w.k + 7) / 8 * 8;                 // rows that begin at 16-byte borders
        out.buf = dev.alloc((size_t)(rows * w.n) * dtype_size(x.dtype), false);
        if (parts > 1) {
            const int64_t tiles = (rows + kSplitRows - 1) / kSplitRows;
            BufferRef split = dev.alloc((size_t)(tiles * 3 * kSplitRows * kp) * 2, false);
            dev.begin_launch("q4_split");
            if (!dev.dry)
                q4_split_kernel<<<grid_for(dev, rows * kp / 8), 256, 0, dev.stream>>>((const float*)x.base_ptr(), x.layout.strides[0], rows, w.k, (__nv_bfloat16*)split->ptr, kp);
            dev.end_launch();
            q4_tc_run(dev, w, tc, split->ptr, DType::BF16, kp, rows, parts, out.base_ptr());
            return out;
        }
        if (kp != w.k || x.layout.strides[0] % 8 || x.layout.strides[0] < w.k || (uintptr_t)x.base_ptr() % 16) {
            TensorData wide;
            wide.dtype = x.dtype;
            wide.layout = Layout::contiguous({rows, kp});
            wide.buf = dev.alloc((size_t)(rows * kp) * dtype_size(x.dtype), false);      // (nothing reads a row behind its last column)
            TensorData window = wide;
            window.layout.shape = {rows, w.k};
            run_copy(dev, window, x);
            x = wide;
        }
        q4_tc_run(dev, w, tc, x.base_ptr(), x.dtype, x.layout.strides[0], rows, parts, out.base_ptr());
        return out;
    }
    if (x.layout.strides[1] != 1 && w.k > 1) x = run_compact(dev, x);
    out.buf = dev.alloc((size_t)(rows * w.n) * dtype_size(x.dtype), false);
    Q4Params p{};
    p.codes = (const uint4*)w.codes->ptr;
    p.scales = w.scales->ptr;
    p.x = x.base_ptr();
    p.x_stride = x.layout.strides[0];
    p.y = out.buf->ptr;
    p.n = w.n;
    p.k = w.k;
    p.rows = plan.block_rows;
    p.all_rows = (int)rows;
    p.columns = plan.block_rows * parts;
    p.chunks = (int)w.chunks;
    p.groups = (int)w.groups;
    p.group_log2 = group_log2(w);
    p.row_tiles = (int)w.row_tiles;
    p.scale_dtype = w.scale_dtype;
    p.tiles = plan.tiles;
    p.share_chunks = (int)((w.chunks + plan.shares - 1) / plan.shares);
    p.aligned = parts == 1 && w.k % 8 == 0 && (rows == 1 || p.x_stride % 8 == 0) && (uintptr_t)p.x % 16 == 0;
    if (x.dtype == DType::F32) dispatch_rows<float>(dev, p, plan.ct, plan.shares);
    else if (x.dtype == DType::F16) dispatch_rows<__half>(dev, p, plan.ct, plan.shares);
    else dispatch_rows<__nv_bfloat16>(dev, p, plan.ct, plan.shares);
    return out;
}

}  // namespace wgf
