// Products with 4-bit weights for many rows, on the tensor cores.
//
//   y[m, n] = sum_k x[m, k] w[n, k],   w[n, k] = scale[n, k / group] * (code[n, k] - 8), rounded once to the type of x
//
// The weights are the A operand: a tile is 128 of their rows by up to 256 rows of x, whose number is chosen so that the tiles
// fill the SMs (q4_tc_plan).  Warp roles of a CTA, one CTA a SM:
//   warp 0       brings x by TMA: 64 columns of all rows of the tile, 128-byte swizzle
//   warp 1       issues tcgen05.mma (M = 128, N = the tile's rows of x, K = 16) into two accumulators in tensor memory in turn
//   warps 2-5    write finished accumulators out: a lane is a row of the weights, so a warp writes 32 neighbours of a row of y
//   warps 6-21   turn codes into the operand: 16 rows by 64 columns are 512 bytes, 16 to a lane, whose words are eight columns in a
//                row of rows g and g + 8 (q4.cu): four 16-byte stores, where the swizzle wants them.  Odd g take the two
//                halves in the other order, so that the lanes of a store fall on different banks.
//   warp 22      brings the codes and scales of two steps at a time by bulk copies
// Every wait is bounded and reports through the device's error word.
//
// Rows of f32 (EXACT): 32 rows of x are three times 32 rows of bf16 parts, which together have their 24 bits; the codes themselves are the
// operand, exactly, and a group's columns have an accumulator of their own, which the epilogue's warps scale and add up in f32 while the
// next ones are made.  500 rows through 4096 x 4096: 138 us with the taking apart, 501 on the warps' own instructions.
//
// What the tiles leave of the last wave is filled by dividing its tiles along the columns: a CTA then leaves its f32 sums in memory, and
// the last of a tile's CTAs adds them up in their order.  64 rows of bf16 through 4096 x 4096: 17 us, 34 undivided; through 4096 x
// 11008: 29, 78 undivided; 500 rows of f16 through 11008 x 4096: 62, 67 undivided (whole tiles alone, of 176 rows), where weights
// written out and the matrix product take 76 together, and the products alone 27 at the measured rate of the tensor cores.
// A step of 64 columns takes 0.4 us with few rows of x and 0.5 with 256, while its products take 0.05 to 0.39: turning the codes into the
// operand, the copies and the handing over of a step cost about 0.2 us each and overlap only in part (without the first 0.33, without
// all of them 0.2), and with 256 rows L2 delivers x at about 9 TB/s.  Tried and not kept (500 rows): 256 rows of weights a tile (half the
// traffic of x: 74 us), two steps to a stage (72), two CTAs a SM with half the decoders (69), one lane that waits for its warp (115).
#include <algorithm>
#include <type_traits>

#include "decode.hpp"
#include "decode_common.cuh"
#include "q4_tc.hpp"
#include "tc_common.cuh"

namespace wgf {

using namespace tc;
using decode::shared_16;
using decode::shared_float2;
using decode::shared_word;

namespace {

constexpr int kBK = 64;                  // columns of a step
constexpr int kDecoders = 16;            // warps; eight have the even steps of a tile and eight the odd ones
constexpr int kThreadsTc = (7 + kDecoders) * 32;
constexpr int kPairs = 4;                // pairs of steps whose codes are on their way
constexpr int kMaxStages = 8;
constexpr int kWBytes = 128 * kBK * 2;   // of a stage: the weights' part
constexpr int kRoom = 225 * 1024;        // shared memory of all stages and pairs

struct Q4TcParams {
    const uint4* codes;
    const void* scales;
    void* y;
    long long n, rows, k;
    int chunks, groups, group_log2, row_tiles;
    DType scale_dtype;
    int tile_rows, out_rows;             // of x, and of y that they make
    int tiles_m, tiles_n, stages;
    int whole, shares, share_chunks;     // tiles of one unit each; units of each of the others, and their steps (an even number)
    float* part;                         // sums of those units: [unit][row of x][128]
    unsigned* tickets;                   // of those tiles
    int scale_bytes, tile_bytes;         // of a scale; of a tile of 16 rows in a pair of steps
    unsigned* error;
};

// A unit of work: a tile, or a share of its steps
struct Unit {
    int tile, share, begin, end;         // share < 0: all of it
    __device__ __forceinline__ Unit(const Q4TcParams& p, int u) {
        tile = u, share = -1, begin = 0, end = p.chunks;
        if (u >= p.whole) {
            tile = p.whole + (u - p.whole) / p.shares;
            share = (u - p.whole) % p.shares;
            begin = share * p.share_chunks;
            end = min(end, begin + p.share_chunks);
            if (p.shares == 1) share = -1;
        }
    }
};

// fp32 accumulator, both operands K-major f16 or bf16, M = 128, N = rows
__device__ __forceinline__ unsigned instruction(bool bf16, int rows) {
    return (1u << 4) | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (unsigned)(rows >> 3) << 17 | (128u >> 4) << 24;
}

// Lanes that give up on a wait take the others of their warp along.
__device__ __forceinline__ bool all_of_warp(bool ok) { return __all_sync(0xffffffffu, ok); }

// What a lane needs of a tile of 16 rows by 64 columns: its words, and as they are stored the scales of rows g and g + 8 for
// each group.  SAME: scales of the type of x, two in a word.
template <bool G32> struct Q4Unit {
    uint4 w;
    uint2 s[G32 ? 2 : 1];
};

// Two codes 16 bits apart as two values of the type, times the scale: code - 8 is exact, the product is rounded once
template <typename T> struct TwoOf;
template <> struct TwoOf<__half> { typedef __half2 type; };
template <> struct TwoOf<__nv_bfloat16> { typedef __nv_bfloat162 type; };
// The nibbles of rows g stand at bit 0 of `nib`, those of rows g + 8 at bit 4.
template <typename T, bool LOW> __device__ __forceinline__ typename TwoOf<T>::type less_eight(unsigned nib) {
    if constexpr (std::is_same<T, __half>::value) {
        const unsigned v = (nib & (LOW ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;          // 1024 + code, or + 16 code
        const __half2 f = *reinterpret_cast<const __half2*>(&v);
        if constexpr (LOW) return __hfma2(f, __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd480)));
        else return __hsub2(f, __half2half2(__ushort_as_half(0x6408)));
    } else {
        const unsigned v = ((LOW ? nib >> 4 : nib) & 0x000f000fu) | 0x43004300u;             // 128 + code
        return __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
    }
}
template <typename T, bool SAME, bool LOW, bool EXACT> __device__ __forceinline__ unsigned two_values(unsigned nib, typename TwoOf<T>::type s2, float s) {
    if constexpr (EXACT) {
        const unsigned v = ((LOW ? nib >> 4 : nib) & 0x000f000fu) | 0x3e003e00u;             // (128 + code) / 1024
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __bfloat162bfloat162(__ushort_as_bfloat16(0x3e08)));
        return *reinterpret_cast<const unsigned*>(&d);
    }
    const auto d = less_eight<T, LOW>(nib);
    if constexpr (SAME) {
        const auto v = __hmul2(d, s2);
        return *reinterpret_cast<const unsigned*>(&v);
    } else {
        return pack2<T>(__low2float(d) * s, __high2float(d) * s);
    }
}
__device__ __forceinline__ __half2 two_low(__half2 v) { return __low2half2(v); }
__device__ __forceinline__ __half2 two_high(__half2 v) { return __high2half2(v); }
__device__ __forceinline__ __nv_bfloat162 two_low(__nv_bfloat162 v) { return __low2bfloat162(v); }
__device__ __forceinline__ __nv_bfloat162 two_high(__nv_bfloat162 v) { return __high2bfloat162(v); }
// The values behind the row's end are zero whatever the scale is
__device__ __forceinline__ uint4 first_of(uint4 v, int valid) {
    unsigned* r = reinterpret_cast<unsigned*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (valid <= 2 * i) r[i] = 0;
        else if (valid == 2 * i + 1) r[i] &= 0xffffu;
    return v;
}
// From global to shared memory, both from 16-byte borders on and in multiples of 16 bytes
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void store16(unsigned at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A unit as the operand.  `at`: the lane's place for the first of the two halves of a row that it writes; the other is 64
// bytes away.  `valid`, where the row ends in the unit (ENDS): columns from the lane's first on in the first half.
template <typename T, bool SAME, bool G32, bool EXACT, bool ENDS>
__device__ __forceinline__ void decode_unit(const Q4Unit<G32>& u, DType scale_dtype, bool odd, unsigned at, int valid) {
    typedef typename TwoOf<T>::type T2;
    const unsigned words[4] = {odd ? u.w.z : u.w.x, odd ? u.w.w : u.w.y, odd ? u.w.x : u.w.z, odd ? u.w.y : u.w.w};
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
        const unsigned a = words[2 * turn], b = words[2 * turn + 1];
        uint2 raw = u.s[0];
        if (G32) raw = (turn == 0) == odd ? u.s[G32 ? 1 : 0] : raw;
        T2 up{}, low{};
        float fu = 0.f, fl = 0.f;
        if constexpr (SAME) {
            const T2 both = *reinterpret_cast<const T2*>(&raw.x);
            up = two_low(both);
            low = two_high(both);
        } else if (scale_dtype == DType::F32) {
            fu = __uint_as_float(raw.x);
            fl = __uint_as_float(raw.y);
        } else if (scale_dtype == DType::F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
            fu = f.x;
            fl = f.y;
        } else {
            fu = __uint_as_float(raw.x << 16);
            fl = __uint_as_float(raw.x & 0xffff0000u);
        }
        const unsigned a8 = a >> 8, b8 = b >> 8;
        uint4 top = make_uint4(two_values<T, SAME, false, EXACT>(a, up, fu), two_values<T, SAME, false, EXACT>(a8, up, fu), two_values<T, SAME, false, EXACT>(b, up, fu),
                               two_values<T, SAME, false, EXACT>(b8, up, fu));
        uint4 bottom = make_uint4(two_values<T, SAME, true, EXACT>(a, low, fl), two_values<T, SAME, true, EXACT>(a8, low, fl), two_values<T, SAME, true, EXACT>(b, low, fl),
                                  two_values<T, SAME, true, EXACT>(b8, low, fl));
        if (ENDS) {
            const int left = valid - 32 * (turn ^ (int)odd);
            top = first_of(top, left);
            bottom = first_of(bottom, left);
        }
        store16(turn ? at ^ 64u : at, top);
        store16((turn ? at ^ 64u : at) + 1024, bottom);
    }
}

// EXACT: x in three parts of bf16, whose 32 rows each are the rows of a tile; the codes are the operand, over 1024, and each group's
// sums are scaled as they are added up, in f32.
template <typename T, bool SAME, bool G32, bool EXACT>
__global__ void __launch_bounds__(kThreadsTc, 1) q4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Q4TcParams p) {
    typedef typename std::conditional<EXACT, float, T>::type Y;
    constexpr int kAccs = EXACT ? 4 : 2, kAccCols = 512 / kAccs;
    extern __shared__ unsigned char smem_raw[];
    __shared__ alignas(8) unsigned long long bars[3 * kMaxStages + 8 + 2 * kPairs];
    __shared__ unsigned tmem_slot, last;
    const unsigned stages_at = (smem_u32(smem_raw) + 1023) & ~1023u;          // the swizzle wants 1024-byte alignment
    const unsigned stage_bytes = kWBytes + (unsigned)p.tile_rows * kBK * 2;
    const unsigned pairs_at = stages_at + p.stages * stage_bytes, pair_bytes = 8u * p.tile_bytes;
    const unsigned bar0 = smem_u32(bars);
    auto x_full = [&](int s) { return bar0 + 8u * s; };
    auto w_full = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
    auto empty = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };
    auto acc_full = [&](int a) { return bar0 + 8u * (3 * kMaxStages + a); };
    auto acc_empty = [&](int a) { return bar0 + 8u * (3 * kMaxStages + 4 + a); };
    auto pair_full = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 8 + b); };
    auto pair_empty = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 8 + kPairs + b); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            mbar_init(x_full(s), 1);
            mbar_init(w_full(s), 8);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < kAccs; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), 4);
        }
        for (int b = 0; b < kPairs; ++b) {
            mbar_init(pair_full(b), 1);
            mbar_init(pair_empty(b), kDecoders);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    const int units = p.whole + (p.tiles_m * p.tiles_n - p.whole) * p.shares;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            unsigned phase = 1;                       // a fresh barrier counts as released
            bool ok = true;
            for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
                const Unit u(p, i);
                const int m0 = u.tile % p.tiles_m * p.tile_rows;
                for (int kb = u.begin; kb < u.end; ++kb) {
                    if (!mbar_wait(empty(stage), phase)) {
                        atomicExch(p.error, 81u);
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(x_full(stage), (unsigned)p.tile_rows * kBK * 2);
                    tma_load_3d(stages_at + stage * stage_bytes + kWBytes, &map_x, x_full(stage), kb * kBK, m0, 0);
                    if (++stage == p.stages) stage = 0, phase ^= 1;
                }
            }
            if (!ok)                                  // what is on its way lands before the CTA ends
                for (int s = 0; s < p.stages; ++s) mbar_wait(x_full(s), s < stage ? phase ^ 1 : phase);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const unsigned idesc = instruction(std::is_same<T, __nv_bfloat16>::value, p.tile_rows);
            const unsigned long long first = smem_desc(stages_at, 16, 1024);      // its addresses are in units of 16 bytes
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 1;
            bool ok = true;
            for (int n = blockIdx.x; n < units && ok; n += gridDim.x) {
                const Unit u(p, n);
                if constexpr (!EXACT) {
                    if (!mbar_wait(acc_empty(acc), acc_phase)) {
                        atomicExch(p.error, 82u);
                        break;
                    }
                    tc_fence_after();
                }
                for (int kb = u.begin; kb < u.end; ++kb) {
                    if (!mbar_wait(x_full(stage), phase) || !mbar_wait(w_full(stage), phase)) {
                        atomicExch(p.error, 83u);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const unsigned long long w = first + (unsigned)stage * (stage_bytes >> 4), x = w + (kWBytes >> 4);
                    if constexpr (EXACT) {
                        const int inside = (1 << p.group_log2) - 1;
                        for (int half = 0; half < 2 && ok; ++half) {
                            const int col = kb * kBK + half * 32;
                            const bool fresh = (col & inside) == 0;
                            if (fresh && !mbar_wait(acc_empty(acc), acc_phase)) {
                                atomicExch(p.error, 82u);
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            umma_f16(tmem + (unsigned)acc * kAccCols, w + 4 * half, x + 4 * half, idesc, !fresh);
                            umma_f16(tmem + (unsigned)acc * kAccCols, w + 4 * half + 2, x + 4 * half + 2, idesc, 1u);
                            if (((col + 32) & inside) == 0 || (half && kb + 1 == u.end)) {
                                umma_commit(acc_full(acc));
                                if (++acc == kAccs) acc = 0, acc_phase ^= 1;
                            }
                        }
                        if (!ok) break;
                    } else {
#pragma unroll
                        for (int i = 0; i < kBK / 16; ++i) umma_f16(tmem + (unsigned)acc * kAccCols, w + 2 * i, x + 2 * i, idesc, kb != u.begin || i != 0);
                    }
                    umma_commit(empty(stage));
                    if (++stage == p.stages) stage = 0, phase ^= 1;
                }
                if constexpr (!EXACT) {
                    if (ok) umma_commit(acc_full(acc));
                    if (++acc == kAccs) acc = 0, acc_phase ^= 1;
                }
            }
        }
    } else if (warp < 6) {
        const int quarter = warp & 3;                 // of the accumulator's lanes
        int acc = 0;
        unsigned acc_phase = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
            const Unit u(p, i);
            const long long m0 = (long long)(u.tile % p.tiles_m) * p.out_rows, n = (long long)(u.tile / p.tiles_m) * 128 + quarter * 32 + lane;
            const int live = (int)min((long long)p.out_rows, p.rows - m0);
            Y* to = (Y*)p.y + m0 * p.n + n;
            float* mine = u.share < 0 ? nullptr : p.part + (long long)(i - p.whole) * p.out_rows * 128 + quarter * 32 + lane;
            // 32 rows of y from c on, of which this lane has column n
            auto put = [&](int c, auto value) {
                if (mine) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c + j < live) mine[(c + j) * 128] = value(j);
                } else if (n < p.n) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c + j < live) to[(c + j) * p.n] = decode::from_f<Y>(value(j));
                }
                __syncwarp();
            };
            const unsigned from = tmem + ((unsigned)(quarter * 32) << 16);
            unsigned v[32];
            if constexpr (EXACT) {
                float sum[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[j] = 0.f;
                const int first = u.begin * kBK >> p.group_log2, end = ((u.end * kBK - 1) >> p.group_log2) + 1;
                const long long row = min(n, (long long)p.row_tiles * 16 - 1), at = (row >> 4) * p.groups * 16 + (row & 7) * 2 + (row >> 3 & 1);
                auto scale = [&](int q) -> float {        // a group behind the last column is all zeros
                    if (q >= p.groups) return 0.f;
                    const long long o = at + q * 16;
                    return p.scale_dtype == DType::F32   ? __ldg((const float*)p.scales + o)
                           : p.scale_dtype == DType::F16 ? __half2float(__ldg((const __half*)p.scales + o))
                                                         : __bfloat162float(__ldg((const __nv_bfloat16*)p.scales + o));
                };
                float ahead = scale(first);
                for (int q = first; q < end; ++q) {
                    const float s = ahead;
                    if (q + 1 < end) ahead = scale(q + 1);
                    if (!all_of_warp(mbar_wait(acc_full(acc), acc_phase))) {
                        if (lane == 0) atomicExch(p.error, 84u);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
                        tmem_ld_32x32(from + (unsigned)(acc * kAccCols + part * 32), v);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[j] = fmaf(__uint_as_float(v[j]), s, sum[j]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty(acc));
                    if (++acc == kAccs) acc = 0, acc_phase ^= 1;
                }
                if (!ok) break;
                put(0, [&](int j) { return sum[j] * 1024.f; });
            } else {
                if (!all_of_warp(mbar_wait(acc_full(acc), acc_phase))) {
                    if (lane == 0) atomicExch(p.error, 84u);
                    break;
                }
                tc_fence_after();
                for (int c = 0; c < live; c += 32) {
                    tmem_ld_32x32(from + (unsigned)(acc * kAccCols + c), v);
                    tmem_ld_wait();
                    put(c, [&](int j) { return __uint_as_float(v[j]); });
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(acc));
                if (++acc == kAccs) acc = 0, acc_phase ^= 1;
            }
        }
    } else if (warp < 6 + kDecoders) {
        const int d = (warp - 6) & 7, odd = (warp - 6) >> 3;
        // where this lane's words, scales and places in the operand are in a pair and a stage
        const unsigned words = pairs_at + d * p.tile_bytes + odd * 512 + lane * 16;
        const unsigned scales = pairs_at + d * p.tile_bytes + 1024 + (((odd * 64) >> p.group_log2) * 16 + (lane >> 2) * 2) * p.scale_bytes;
        const int g = lane >> 2, c = lane & 3;
        const unsigned operand = stages_at + (d * 16 + g) * 128 + (((g & 1) * 4 + c) ^ g) * 16;
        int stage = 0, buffer = 0;
        unsigned phase = 1, pair_phase = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
            const Unit work(p, i);
            for (int kb = work.begin; kb < work.end; kb += 2) {
                int s = stage + odd;
                unsigned s_phase = phase;
                if (s >= p.stages) s -= p.stages, s_phase ^= 1;
                const bool live = kb + odd < work.end;
                if (!all_of_warp(mbar_wait(pair_full(buffer), pair_phase) && (!live || mbar_wait(empty(s), s_phase)))) {
                    if (lane == 0) atomicExch(p.error, 85u);
                    ok = false;
                    break;
                }
                if (live) {
                    Q4Unit<G32> u;
                    u.w = shared_16(words + buffer * pair_bytes);
#pragma unroll
                    for (int i = 0; i < (G32 ? 2 : 1); ++i) {
                        const unsigned at = scales + buffer * pair_bytes + i * 16 * p.scale_bytes;
                        if (!SAME && p.scale_bytes == 4) {
                            const float2 f = shared_float2(at);
                            u.s[i] = make_uint2(__float_as_uint(f.x), __float_as_uint(f.y));
                        } else {
                            u.s[i].x = shared_word(at);
                        }
                    }
                    const unsigned at = operand + s * stage_bytes;
                    const int valid = (int)p.k - (kb + odd) * kBK - c * 8;
                    if (valid + c * 8 >= kBK) decode_unit<T, SAME, G32, EXACT, false>(u, p.scale_dtype, g & 1, at, valid);
                    else decode_unit<T, SAME, G32, EXACT, true>(u, p.scale_dtype, g & 1, at, valid);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) {
                    if (live) mbar_arrive(w_full(s));
                    mbar_arrive(pair_empty(buffer));
                }
                stage += min(2, work.end - kb);
                if (stage >= p.stages) stage -= p.stages, phase ^= 1;
                if (++buffer == kPairs) buffer = 0, pair_phase ^= 1;
            }
        }
    } else {
        int buffer = 0;
        unsigned phase = 1;
        bool ok = true;
        for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
            const Unit u(p, i);
            // tiles behind the last are the last again: nobody reads what becomes of their rows
            const long long rt = min(u.tile / p.tiles_m * 8 + (lane & 7), p.row_tiles - 1);
            const uint4* words = p.codes + rt * p.chunks * 32;
            const unsigned char* scales = (const unsigned char*)p.scales + rt * p.groups * 16 * p.scale_bytes;
            for (int kb = u.begin; kb < u.end; kb += 2) {
                if (!all_of_warp(mbar_wait(pair_empty(buffer), phase))) {
                    if (lane == 0) atomicExch(p.error, 86u);
                    ok = false;
                    break;
                }
                const int q = kb * 64 >> p.group_log2;
                const unsigned wb = min(2, u.end - kb) * 512u, sb = min(128 >> p.group_log2, p.groups - q) * 16u * p.scale_bytes;
                if (lane == 0) mbar_expect_tx(pair_full(buffer), 8 * (wb + sb));
                __syncwarp();
                if (lane < 8) {
                    const unsigned to = pairs_at + buffer * pair_bytes + lane * p.tile_bytes;
                    bulk_load(to, words + kb * 32, wb, pair_full(buffer));
                    bulk_load(to + 1024, scales + q * 16 * p.scale_bytes, sb, pair_full(buffer));
                }
                if (++buffer == kPairs) buffer = 0, phase ^= 1;
            }
        }
        if (!ok)
            for (int b = 0; b < kPairs; ++b) mbar_wait(pair_full(b), b < buffer ? phase ^ 1 : phase);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    // A CTA has at most one share of a tile, its last unit.  The last CTA of a tile's adds up what all have left, in their order.
    if (p.shares == 1) return;
    const int i = blockIdx.x + (units - 1 - blockIdx.x) / gridDim.x * gridDim.x;
    if (i < p.whole) return;
    const Unit u(p, i);
    if (threadIdx.x == 0) {
        __threadfence();                                       // behind the barrier: for all that the CTA has written
        last = atomicAdd(p.tickets + (u.tile - p.whole), 1u) == (unsigned)p.shares - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    const long long m0 = (long long)(u.tile % p.tiles_m) * p.out_rows, n0 = (long long)(u.tile / p.tiles_m) * 128 + lane * 4;
    const int live = (int)min((long long)p.out_rows, p.rows - m0);
    const float* parts = p.part + (long long)(u.tile - p.whole) * p.shares * p.out_rows * 128 + lane * 4;
    for (int c = warp; c < live; c += kThreadsTc / 32) {       // a warp has whole rows of x
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < p.shares; ++s) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + ((long long)s * p.out_rows + c) * 128));
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
        Y* row = (Y*)p.y + (m0 + c) * p.n + n0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n0 + e < p.n) row[e] = decode::from_f<Y>(f[e]);
    }
    if (threadIdx.x == 0) p.tickets[u.tile - p.whole] = 0;
}

}  // namespace

// Tiles of few rows of x cost nearly what tiles of many do, as the time goes into the weights' side: so as few waves as 256 rows
// allow.  The tiles of the last wave are divided along the columns, where the SMs that they leave would wait, if the adding up
// costs less.  In us: a step of 64 columns takes 0.44 with 64 rows of x, 0.47 with 128, 0.55 with 256; adding up 2.5, and 0.0105 for
// each row of x in each share.  Rows of f32: 0.5, with groups of 32 (four accumulators for two steps) 0.8.
Q4TcPlan q4_tc_plan(Device& dev, const Q4Weight& w, int64_t rows, bool exact) {
    Q4TcPlan best;
    const int64_t tiles_n = (w.row_tiles + 7) / 8, most_rows = exact ? kExactRows : 256, least = (rows + most_rows - 1) / most_rows, sms = dev.sm_count;
    int64_t before = 0;
    for (int64_t t = least; t < least + (exact ? 1 : 8); ++t) {
        const int64_t tile_rows = exact ? kExactRows : ((rows + t - 1) / t + 15) / 16 * 16;
        if (tile_rows == before) continue;
        before = tile_rows;
        const int64_t tiles = tiles_n * ((rows + tile_rows - 1) / tile_rows), whole = tiles / sms * sms, rest = tiles - whole;
        const double step = exact ? (w.group == 32 ? 0.8 : 0.5) : 0.40 + 0.0006 * (double)tile_rows, start = 5.0 + (double)(whole / sms * w.chunks) * step;
        const int most = rest ? (int)std::min<int64_t>(sms / rest, 32) : 1;      // a CTA has one share at most
        for (int s = 1; s <= most; ++s) {
            const int steps = s == 1 ? (int)w.chunks : (((int)w.chunks + s - 1) / s + 1) / 2 * 2, shares = ((int)w.chunks + steps - 1) / steps;
            if (shares < s) continue;
            const double us = start + (rest ? (double)steps * step : 0) + (shares > 1 ? 2.5 + 0.0105 * (double)(shares * tile_rows) : 0);
            if (us < best.us) best = {(int)tile_rows, (int)whole, shares, steps, us};
        }
    }
    return best;
}

bool q4_tc_run(Device& dev, const Q4Weight& w, const Q4TcPlan& plan, const void* x, DType dtype, int64_t stride, int64_t rows, bool exact, void* y) {
    const bool bf16 = dtype == DType::BF16;
    const int tile_rows = exact ? 3 * plan.tile_rows : plan.tile_rows;
    const int64_t x_rows = exact ? (rows + kExactRows - 1) / kExactRows * tile_rows : rows;
    if (x_rows >= (1ll << 31) - 256) return false;            // coordinates of TMA are 32 bits
    CUtensorMap map;
    if (!dev.dry && !encode_3d(&map, bf16, x, w.k, x_rows, 1, stride, x_rows * stride, kBK, (unsigned)tile_rows)) return false;
    Q4TcParams p{};
    p.codes = (const uint4*)w.codes->ptr;
    p.scales = w.scales->ptr;
    p.y = y;
    p.n = w.n;
    p.rows = rows;
    p.k = w.k;
    p.chunks = (int)w.chunks;
    p.groups = (int)w.groups;
    p.group_log2 = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    p.row_tiles = (int)w.row_tiles;
    p.scale_dtype = w.scale_dtype;
    p.tile_rows = tile_rows;
    p.out_rows = plan.tile_rows;
    p.tiles_m = (int)((rows + plan.tile_rows - 1) / plan.tile_rows);
    p.tiles_n = (int)((w.row_tiles + 7) / 8);
    p.scale_bytes = (int)dtype_size(w.scale_dtype);
    p.tile_bytes = 1024 + (int)(128 / w.group) * 16 * p.scale_bytes;
    const int stage_bytes = kWBytes + tile_rows * kBK * 2, pairs_bytes = kPairs * 8 * p.tile_bytes;
    p.stages = std::min(kMaxStages, (kRoom - pairs_bytes) / stage_bytes);
    p.error = dev.error_word();
    p.whole = plan.whole;
    p.shares = plan.shares;
    p.share_chunks = plan.share_chunks;
    const int64_t divided = (int64_t)p.tiles_m * p.tiles_n - p.whole;     // fewer than SMs
    BufferRef scratch;
    if (p.shares > 1) {
        scratch = dev.alloc((size_t)(divided * p.shares * p.out_rows) * 128 * sizeof(float), false);
        p.part = (float*)scratch->ptr;
        p.tickets = (unsigned*)dev.counters();
    }
    const unsigned grid = (unsigned)std::min<int64_t>(p.whole + divided * p.shares, dev.sm_count);
    const int smem = p.stages * stage_bytes + pairs_bytes + 1024;
    dev.begin_launch("q4_tc");
    if (!dev.dry) {
        auto go = [&](auto kernel) {
            WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom + 1024));
            kernel<<<grid, kThreadsTc, smem, dev.stream>>>(map, p);
        };
        const bool same = w.scale_dtype == dtype, g32 = w.group == 32;
        if (exact) {
            go(q4_tc_kernel<__nv_bfloat16, false, false, true>);
        } else if (bf16) {
            if (same) g32 ? go(q4_tc_kernel<__nv_bfloat16, true, true, false>) : go(q4_tc_kernel<__nv_bfloat16, true, false, false>);
            else g32 ? go(q4_tc_kernel<__nv_bfloat16, false, true, false>) : go(q4_tc_kernel<__nv_bfloat16, false, false, false>);
        } else {
            if (same) g32 ? go(q4_tc_kernel<__half, true, true, false>) : go(q4_tc_kernel<__half, true, false, false>);
            else g32 ? go(q4_tc_kernel<__half, false, true, false>) : go(q4_tc_kernel<__half, false, false, false>);
        }
    }
    dev.end_launch();
    return true;
}

}  // namespace wgf
