// Products with 4-bit weights for many rows, on the tensor cores.
//
//   y[m, n] = sum over groups of columns of scale[n, group] * sum_{k in group} x[m, k] * (code[n, k] - 8)
//
// The codes less 8 are the A operand, exactly, and the rows of x the B operand: every product is exact, a group's columns have an accumulator
// of their own, and the scale enters in f32 when the group's sum is added to the others.  Rounded are f32 sums, and y once.  (Weights that are
// rounded to 16 bits on the way would need neither the accumulators nor the adding up; for f16 the result's error is then a quarter larger.)
//
// A tile is 128 rows of the weights by up to 256 rows of x, whose number is chosen so that the tiles fill the SMs (q4_tc_plan).  Warp roles of a CTA,
// one CTA a SM:
//   warp 0        brings x by TMA: 64 columns of all rows of the tile, 128-byte swizzle
//   warp 1        issues tcgen05.mma (M = 128, N = the tile's rows of x, K = 16) into two or four accumulators in tensor memory in turn
//   warp 2        brings the codes of two steps at a time by bulk copies
//   warps 4-11    scale and add up finished groups, in registers: a lane is a row of the weights, four warps have the first half of the rows of x
//                 and four the second; at the tile's end a warp writes 32 neighbours of a row of y
//   warps 12-19   turn codes into the operand: 16 rows by 64 columns are 512 bytes, 16 to a lane, whose words are eight columns in a
//                 row of rows g and g + 8 (q4.cu): four 16-byte stores, where the swizzle wants them.  Odd g take the two
//                 halves in the other order, so that the lanes of a store fall on different banks.
// The sums of 128 rows of x are 128 registers a lane; the other warps leave theirs to those that add up.
// Every wait is bounded and reports through the device's error word.
//
// Rows of f32: 32 rows of x are three times 32 rows of bf16 parts, which together have their 24 bits, and are added up as if they were more columns.
//
// What the tiles leave of the last wave is filled by dividing its tiles along the columns: a CTA then leaves its f32 sums in memory, and
// the last of a tile's CTAs adds them up in their order, eight rows side by side (a row after the other took 27 us for six shares of 250 rows, eight 2).
//
// 500 rows of f16 through 11008 x 4096: 62 us with groups of 128, 68 with groups of 64, 109 with groups of 32; 64 rows of bf16 through 4096 x 4096: 17;
// 500 rows of f32 through 4096 x 4096: 145 with the taking apart.  The products alone would take 27 for the first at the measured rate of the tensor cores.
// With groups of 128 x bounds it: 32 KB a step for every SM are 9 TB/s from L2.  With shorter groups the adding up does, whose warps wait for what they
// read from tensor memory: 176 registers hold 128 sums and 32 columns on their way (16 at a time: 72 and 112).  Scales stay as they are stored until they
// are used: converted where they were called for, each fourth group waited for memory (81 with groups of 64).  A step with few rows takes 0.45
// us, by time stamps nearly all of it the issuing lane's waits and commits one after the other; its products are 0.07.
#include <algorithm>
#include <type_traits>

#include "decode.hpp"
#include "decode_common.cuh"
#include "q4_tc.hpp"
#include "tc_common.cuh"

namespace wgf {

using namespace tc;
using decode::shared_16;

namespace {

constexpr int kBK = 64;                  // columns of a step
constexpr int kAdders = 8, kDecoders = 8;                      // warps
constexpr int kFirstAdder = 4, kFirstDecoder = kFirstAdder + kAdders;
constexpr int kThreadsTc = (kFirstDecoder + kDecoders) * 32;
// Registers: what the CTA starts with is shared out anew, and no more than that.
constexpr int kStartRegs = 96, kAdderRegs = 176, kOtherRegs = 40;
static_assert(kAdders * kAdderRegs + (kThreadsTc / 32 - kAdders) * kOtherRegs <= kThreadsTc / 32 * kStartRegs, "more registers than the CTA has");
constexpr int kPairs = 4;                // pairs of steps whose codes are on their way
constexpr int kMaxStages = 8, kMaxAccs = 4;
constexpr int kWBytes = 128 * kBK * 2;   // of a stage: the weights' part
constexpr int kPairBytes = 8 * 1024;     // codes of 128 rows by 128 columns
constexpr int kRoom = 225 * 1024;        // shared memory of all stages and pairs

struct Q4TcParams {
    const uint4* codes;
    const void* scales;
    void* y;
    long long n, rows;
    int chunks, groups, group_log2, row_tiles;
    DType scale_dtype;
    int tile_rows, out_rows;             // of x, and of y that they make
    int accs;                            // accumulators: two of 256 columns or four of 128
    int tiles_m, tiles_n, stages;
    int whole, shares, share_chunks;     // tiles of one unit each; units of each of the others, and their steps (an even number)
    float* part;                         // sums of those units: [unit][row of x][128]
    unsigned* tickets;                   // of those tiles
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

// Two codes 16 bits apart as two values of the type, exactly: code - 8 as f16, and (code - 8) / 1024 as bf16, whose x may be anywhere in the
// range of f32, which sums of 128 products must not leave.  The nibbles of rows g stand at bit 0 of `nib`, those of rows g + 8 at bit 4.
template <typename T> __device__ __forceinline__ float operand_unit() { return std::is_same<T, __half>::value ? 1.f : 1024.f; }
template <typename T, bool LOW> __device__ __forceinline__ unsigned less_eight(unsigned nib) {
    if constexpr (std::is_same<T, __half>::value) {
        const unsigned v = (nib & (LOW ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;          // 1024 + code, or + 16 code
        const __half2 f = *reinterpret_cast<const __half2*>(&v);
        __half2 d;
        if constexpr (LOW) d = __hfma2(f, __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd480)));
        else d = __hsub2(f, __half2half2(__ushort_as_half(0x6408)));
        return *reinterpret_cast<const unsigned*>(&d);
    } else {
        const unsigned v = ((LOW ? nib >> 4 : nib) & 0x000f000fu) | 0x3e003e00u;             // (128 + code) / 1024
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __bfloat162bfloat162(__ushort_as_bfloat16(0x3e08)));
        return *reinterpret_cast<const unsigned*>(&d);
    }
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
__device__ __forceinline__ void tmem_ld_32x16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
// Two f32 sums side by side: sum += a * b
__device__ __forceinline__ void add_two(unsigned long long& sum, unsigned lo, unsigned hi, unsigned long long b) {
    const unsigned long long a = (unsigned long long)hi << 32 | lo;
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(a), "l"(b));
}
template <int N> __device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void leave_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void adders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kAdders * 32) : "memory"); }

// A lane's words of 16 rows by 64 columns as the operand.  `at`: its place for the first of the two halves of a row that it writes; the other is 64 bytes
// away.  Columns behind the end of the weights have codes of zero, and x is zero there.
template <typename T> __device__ __forceinline__ void decode_unit(uint4 w, bool odd, unsigned at) {
    const unsigned words[4] = {odd ? w.z : w.x, odd ? w.w : w.y, odd ? w.x : w.z, odd ? w.y : w.w};
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
        const unsigned a = words[2 * turn], b = words[2 * turn + 1], a8 = a >> 8, b8 = b >> 8;
        const unsigned to = turn ? at ^ 64u : at;
        store16(to, make_uint4(less_eight<T, false>(a), less_eight<T, false>(a8), less_eight<T, false>(b), less_eight<T, false>(b8)));
        store16(to + 1024, make_uint4(less_eight<T, true>(a), less_eight<T, true>(a8), less_eight<T, true>(b), less_eight<T, true>(b8)));
    }
}

// PARTS: 1, or 3 for rows of f32, whose bf16 parts, 32 rows each, are the rows of a tile.
template <typename T, int PARTS>
__global__ void __launch_bounds__(kThreadsTc, 1) q4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Q4TcParams p) {
    typedef typename std::conditional<PARTS == 1, T, float>::type Y;
    extern __shared__ unsigned char smem_raw[];
    __shared__ alignas(8) unsigned long long bars[3 * kMaxStages + 2 * kMaxAccs + 2 * kPairs];
    __shared__ unsigned tmem_slot, last;
    const unsigned stages_at = (smem_u32(smem_raw) + 1023) & ~1023u;          // the swizzle wants 1024-byte alignment
    const unsigned stage_bytes = kWBytes + (unsigned)p.tile_rows * kBK * 2;
    const unsigned pairs_at = stages_at + p.stages * stage_bytes;
    const unsigned bar0 = smem_u32(bars);
    auto x_full = [&](int s) { return bar0 + 8u * s; };
    auto w_full = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
    auto empty = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };
    auto acc_full = [&](int a) { return bar0 + 8u * (3 * kMaxStages + a); };
    auto acc_empty = [&](int a) { return bar0 + 8u * (3 * kMaxStages + kMaxAccs + a); };
    auto pair_full = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 2 * kMaxAccs + b); };
    auto pair_empty = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 2 * kMaxAccs + kPairs + b); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            mbar_init(x_full(s), 1);
            mbar_init(w_full(s), kDecoders);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < kMaxAccs; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), kAdders);
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
    const unsigned tmem = tmem_slot, acc_columns = 512u / (unsigned)p.accs;
    const int units = p.whole + (p.tiles_m * p.tiles_n - p.whole) * p.shares;

    if (warp < kFirstAdder) {
        leave_registers<kOtherRegs>();
        if (warp == 0 && lane == 0) {
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
        } else if (warp == 1 && lane == 0) {
            const unsigned idesc = instruction(std::is_same<T, __nv_bfloat16>::value, p.tile_rows);
            const unsigned long long first = smem_desc(stages_at, 16, 1024);      // its addresses are in units of 16 bytes
            const int inside = (1 << p.group_log2) - 1;
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 1;
            bool ok = true;
            for (int n = blockIdx.x; n < units && ok; n += gridDim.x) {
                const Unit u(p, n);
                for (int kb = u.begin; kb < u.end; ++kb) {
                    if (!mbar_wait(x_full(stage), phase) || !mbar_wait(w_full(stage), phase)) {
                        atomicExch(p.error, 83u);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const unsigned long long w = first + (unsigned)stage * (stage_bytes >> 4), x = w + (kWBytes >> 4);
                    for (int half = 0; half < 2; ++half) {
                        const int col = kb * kBK + half * 32;
                        const bool fresh = (col & inside) == 0;
                        if (fresh) {
                            if (!mbar_wait(acc_empty(acc), acc_phase)) {
                                atomicExch(p.error, 82u);
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                        }
                        umma_f16(tmem + (unsigned)acc * acc_columns, w + 4 * half, x + 4 * half, idesc, !fresh);
                        umma_f16(tmem + (unsigned)acc * acc_columns, w + 4 * half + 2, x + 4 * half + 2, idesc, 1u);
                        if (((col + 32) & inside) == 0 || (half && kb + 1 == u.end)) {
                            umma_commit(acc_full(acc));
                            if (++acc == p.accs) acc = 0, acc_phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    umma_commit(empty(stage));
                    if (++stage == p.stages) stage = 0, phase ^= 1;
                }
            }
        } else if (warp == 2) {
            int buffer = 0;
            unsigned phase = 1;
            bool ok = true;
            for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
                const Unit u(p, i);
                // tiles behind the last are the last again: nobody reads what becomes of their rows
                const long long rt = min(u.tile / p.tiles_m * 8 + (lane & 7), p.row_tiles - 1);
                const uint4* words = p.codes + rt * p.chunks * 32;
                for (int kb = u.begin; kb < u.end; kb += 2) {
                    if (!all_of_warp(mbar_wait(pair_empty(buffer), phase))) {
                        if (lane == 0) atomicExch(p.error, 86u);
                        ok = false;
                        break;
                    }
                    const unsigned bytes = min(2, u.end - kb) * 512u;
                    if (lane == 0) mbar_expect_tx(pair_full(buffer), 8 * bytes);
                    __syncwarp();
                    if (lane < 8) bulk_load(pairs_at + buffer * kPairBytes + lane * 1024, words + kb * 32, bytes, pair_full(buffer));
                    if (++buffer == kPairs) buffer = 0, phase ^= 1;
                }
            }
            if (!ok)
                for (int b = 0; b < kPairs; ++b) mbar_wait(pair_full(b), b < buffer ? phase ^ 1 : phase);
        }
        __syncwarp();
        tc_fence_before();
        __syncthreads();
        if (warp == 1) {
            tc_fence_after();
            tmem_dealloc(tmem, 512);
        }
    } else if (warp >= kFirstDecoder) {
        leave_registers<kOtherRegs>();
        // where this lane's words and its places in the operand are in a pair and a stage
        const int d = warp - kFirstDecoder, g = lane >> 2, c = lane & 3;
        const unsigned words = pairs_at + d * 1024 + lane * 16;
        const unsigned operand = stages_at + (d * 16 + g) * 128 + (((g & 1) * 4 + c) ^ g) * 16;
        int stage = 0, buffer = 0;
        unsigned phase = 1, pair_phase = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
            const Unit u(p, i);
            for (int kb = u.begin; kb < u.end && ok; kb += 2) {
                ok = all_of_warp(mbar_wait(pair_full(buffer), pair_phase));
                if (!ok) break;
                uint4 w[2];
                w[0] = shared_16(words + buffer * kPairBytes);
                w[1] = kb + 1 < u.end ? shared_16(words + buffer * kPairBytes + 512) : make_uint4(0, 0, 0, 0);
                __syncwarp();
                if (lane == 0) mbar_arrive(pair_empty(buffer));
                if (++buffer == kPairs) buffer = 0, pair_phase ^= 1;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (kb + s >= u.end) break;
                    ok = all_of_warp(mbar_wait(empty(stage), phase));
                    if (!ok) break;
                    decode_unit<T>(w[s], g & 1, operand + stage * stage_bytes);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(w_full(stage));
                    if (++stage == p.stages) stage = 0, phase ^= 1;
                }
            }
        }
        if (!ok && lane == 0) atomicExch(p.error, 85u);
        tc_fence_before();
        __syncthreads();
    } else {
        take_registers<kAdderRegs>();
        constexpr int kRows = PARTS == 1 ? 128 : 16;      // of x, that a lane adds up
        constexpr int kPieces = PARTS == 1 ? kRows / 32 : PARTS;
        const int quarter = warp & 3, half = (warp - kFirstAdder) >> 2;       // of the accumulator's lanes, of the rows of x
        const int rows = PARTS == 1 ? p.tile_rows / 2 : kRows;
        const unsigned from = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(half * rows);
        int acc = 0;
        unsigned acc_phase = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < units && ok; i += gridDim.x) {
            const Unit u(p, i);
            const long long n = (long long)(u.tile / p.tiles_m) * 128 + quarter * 32 + lane;
            unsigned long long sum[kRows / 2];
#pragma unroll
            for (int j = 0; j < kRows / 2; ++j) sum[j] = 0;
            const int first = u.begin * kBK >> p.group_log2, end = ((u.end * kBK - 1) >> p.group_log2) + 1;
            const long long row = min(n, (long long)p.row_tiles * 16 - 1), at = (row >> 4) * p.groups * 16 + (row & 7) * 2 + (row >> 3 & 1);
            // scales are called for, as they are stored, two groups before they are used; a group behind the last column is all zeros
            auto scale = [&](int q) -> unsigned {
                if (q >= p.groups) return 0u;
                const long long o = at + q * 16ll;
                return p.scale_dtype == DType::F32 ? __ldg((const unsigned*)p.scales + o) : (unsigned)__ldg((const unsigned short*)p.scales + o);
            };
            unsigned ahead[2] = {scale(first), scale(first + 1)};
#pragma unroll 1
            for (int q = first; q < end && ok; q += 2) {
#pragma unroll 1
                for (int e = 0; e < 2 && q + e < end; ++e) {
                    const unsigned raw = e == 0 ? ahead[0] : ahead[1];
                    if (e == 0) ahead[0] = scale(q + 2);
                    else ahead[1] = scale(q + 3);
                    const float s = p.scale_dtype == DType::F32   ? __uint_as_float(raw)
                                    : p.scale_dtype == DType::F16 ? __half2float(__ushort_as_half((unsigned short)raw))
                                                                  : __uint_as_float(raw << 16);
                    const unsigned long long s2 = (unsigned long long)__float_as_uint(s) << 32 | __float_as_uint(s);
                    ok = all_of_warp(mbar_wait(acc_full(acc), acc_phase));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < kPieces; ++c) {
                        constexpr int W = PARTS == 1 ? 32 : 16;
                        if (PARTS == 1 && c * W >= rows) break;
                        unsigned v[W];
                        if constexpr (PARTS == 1) tmem_ld_32x32(from + (unsigned)acc * acc_columns + c * 32, v);
                        else tmem_ld_32x16(from + (unsigned)acc * acc_columns + c * 32, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < W / 2; ++j) add_two(sum[(PARTS == 1 ? c * W / 2 : 0) + j], v[2 * j], v[2 * j + 1], s2);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty(acc));
                    if (++acc == p.accs) acc = 0, acc_phase ^= 1;
                }
            }
            if (!ok) break;
            // the lane's rows of y, of which it has column n
            const long long m0 = (long long)(u.tile % p.tiles_m) * p.out_rows + half * rows;
            const int live = (int)min((long long)rows, p.rows - m0);
            auto value = [&](int j) { return __uint_as_float(j & 1 ? (unsigned)(sum[j / 2] >> 32) : (unsigned)sum[j / 2]) * operand_unit<T>(); };
            if (u.share >= 0) {
                float* mine = p.part + ((long long)(i - p.whole) * p.out_rows + half * rows) * 128 + quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < kRows; ++j)
                    if (j < live) mine[j * 128] = value(j);
            } else if (PARTS == 1 && p.n % 2 == 0) {
                // two lanes side by side exchange values: one writes both columns of a row, the other those of the next
                const bool odd = lane & 1;
                const bool mine = (n & ~1ll) < p.n;
                T* to = (T*)p.y + (m0 + odd) * p.n + (n & ~1ll);
#pragma unroll
                for (int j = 0; j < kRows; j += 2) {
                    const float a = value(j), b = value(j + 1), other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
                    const unsigned both = pack2<T>(odd ? other : a, odd ? b : other);
                    if (mine && j + odd < live) *reinterpret_cast<unsigned*>(to) = both;
                    to += 2 * p.n;
                }
            } else if (n < p.n) {
                Y* to = (Y*)p.y + m0 * p.n + n;
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (j < live) *to = decode::from_f<Y>(value(j));
                    to += p.n;
                }
            }
        }
        if (!ok && lane == 0) atomicExch(p.error, 84u);
        tc_fence_before();
        __syncthreads();
        // A CTA has at most one share of a tile, its last unit.  The last CTA of a tile's adds up what all have left, in their order.
        const int i = blockIdx.x + (units - 1 - blockIdx.x) / gridDim.x * gridDim.x;
        if (p.shares > 1 && i >= p.whole) {
            const Unit u(p, i);
            if (threadIdx.x == kFirstAdder * 32) {
                __threadfence();                                   // behind the barrier: for all that the CTA has written
                last = atomicAdd(p.tickets + (u.tile - p.whole), 1u) == (unsigned)p.shares - 1;
                __threadfence();
            }
            adders_sync();
            if (last) {
                const long long m0 = (long long)(u.tile % p.tiles_m) * p.out_rows, n0 = (long long)(u.tile / p.tiles_m) * 128 + lane * 4;
                const int live = (int)min((long long)p.out_rows, p.rows - m0);
                const float* parts = p.part + (long long)(u.tile - p.whole) * p.shares * p.out_rows * 128 + lane * 4;
                constexpr int kAtOnce = 8;                                     // rows of x that a warp adds up side by side
                for (int c0 = warp - kFirstAdder; c0 < live; c0 += kAdders * kAtOnce) {
                    float4 sum[kAtOnce];
#pragma unroll
                    for (int r = 0; r < kAtOnce; ++r) sum[r] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                    for (int s = 0; s < p.shares; ++s)
#pragma unroll
                        for (int r = 0; r < kAtOnce; ++r) {
                            const int c = min(c0 + r * kAdders, live - 1);
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + ((long long)s * p.out_rows + c) * 128));
                            sum[r].x += v.x, sum[r].y += v.y, sum[r].z += v.z, sum[r].w += v.w;
                        }
#pragma unroll
                    for (int r = 0; r < kAtOnce; ++r) {
                        const int c = c0 + r * kAdders;
                        const float f[4] = {sum[r].x, sum[r].y, sum[r].z, sum[r].w};
                        Y* row = (Y*)p.y + (m0 + c) * p.n + n0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c < live && n0 + e < p.n) row[e] = decode::from_f<Y>(f[e]);
                    }
                }
                if (threadIdx.x == kFirstAdder * 32) p.tickets[u.tile - p.whole] = 0;
            }
        }
    }
}

}  // namespace

// Tiles of few rows of x cost nearly what tiles of many do, as the time goes into the weights' side: so as few waves as 256 rows
// allow.  The tiles of the last wave are divided along the columns, where the SMs that they leave would wait, if the adding up
// costs less.  In us: a step of 64 columns takes 0.49 with 64 rows of x and 0.63 with 256 where groups are of 128 columns, 0.03 more where they are
// shorter, and as long as its groups' adding up where that takes longer (0.66 a group with 256 rows); joining shares 2.5, and 0.007 for each row of x in
// each share.  Rows of f32: 0.50 a step with groups of 128, 0.58 with groups of 64, 0.80 with groups of 32.  Estimated / measured, f16: 11008 x 4096,
// groups of 128, 9 / 64 / 500 rows 34.5 / 38.0, 36.6 / 38.4, 65 / 62; 4096 x 11008, groups of 64, 64 / 500 rows 33 / 34, 71 / 68.
Q4TcPlan q4_tc_plan(Device& dev, const Q4Weight& w, int64_t rows, int parts) {
    Q4TcPlan best;
    const bool split = parts > 1;
    const int64_t tiles_n = (w.row_tiles + 7) / 8, most_rows = split ? kSplitRows : 256, least = (rows + most_rows - 1) / most_rows, sms = dev.sm_count;
    int64_t before = 0;
    for (int64_t t = least; t < least + (split ? 1 : 8); ++t) {
        const int64_t tile_rows = split ? kSplitRows : ((rows + t - 1) / t + 15) / 16 * 16;
        if (tile_rows == before) continue;
        before = tile_rows;
        const int64_t tiles = tiles_n * ((rows + tile_rows - 1) / tile_rows), whole = tiles / sms * sms, rest = tiles - whole;
        const double step = split ? (w.group == 32 ? 0.80 : w.group == 64 ? 0.58 : 0.50)
                                  : std::max((w.group == 128 ? 0.45 : 0.48) + 0.0007 * (double)tile_rows, (0.10 + 0.0022 * (double)tile_rows) * 64.0 / (double)w.group);
        const double start = 5.0 + (double)(whole / sms * w.chunks) * step;
        const int most = rest ? (int)std::min<int64_t>(sms / rest, 32) : 1;      // a CTA has one share at most
        for (int s = 1; s <= most; ++s) {
            const int steps = s == 1 ? (int)w.chunks : (((int)w.chunks + s - 1) / s + 1) / 2 * 2, shares = ((int)w.chunks + steps - 1) / steps;
            if (shares < s) continue;
            const double us = start + (rest ? (double)steps * step : 0) + (shares > 1 ? 2.5 + 0.007 * (double)(shares * tile_rows) : 0);
            if (us < best.us) best = {(int)tile_rows, (int)whole, shares, steps, us};
        }
    }
    return best;
}

void q4_tc_run(Device& dev, const Q4Weight& w, const Q4TcPlan& plan, const void* x, DType dtype, int64_t stride, int64_t rows, int parts, void* y) {
    const int tile_rows = parts * plan.tile_rows;
    const int64_t x_rows = parts > 1 ? (rows + kSplitRows - 1) / kSplitRows * tile_rows : rows;
    WGF_CHECK(x_rows < (1ll << 31) - 256, WGF_ERR_UNSUPPORTED, "too many rows for one product with 4-bit weights");     // coordinates of TMA are 32 bits
    CUtensorMap map;
    if (!dev.dry && !encode_3d(&map, dtype == DType::BF16, x, w.k, x_rows, 1, stride, x_rows * stride, kBK, (unsigned)tile_rows))
        fail(WGF_ERR_CUDA, "the rows of a product with 4-bit weights cannot be described to TMA");
    Q4TcParams p{};
    p.codes = (const uint4*)w.codes->ptr;
    p.scales = w.scales->ptr;
    p.y = y;
    p.n = w.n;
    p.rows = rows;
    p.chunks = (int)w.chunks;
    p.groups = (int)w.groups;
    p.group_log2 = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    p.row_tiles = (int)w.row_tiles;
    p.scale_dtype = w.scale_dtype;
    p.tile_rows = tile_rows;
    p.out_rows = plan.tile_rows;
    p.accs = tile_rows <= 128 ? 4 : 2;
    p.tiles_m = (int)((rows + plan.tile_rows - 1) / plan.tile_rows);
    p.tiles_n = (int)((w.row_tiles + 7) / 8);
    const int stage_bytes = kWBytes + tile_rows * kBK * 2, pairs_bytes = kPairs * kPairBytes;
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
    auto go = [&](auto kernel, int which) {
        if (!dev.dry) {
            static unsigned long long done[3];     // one bit a device; setting it twice does no harm
            if (dev.ordinal >= 64 || !(done[which] >> dev.ordinal & 1)) {
                // the adders wait for registers that the others leave: there have to be as many as the split counts on
                cudaFuncAttributes a;
                WGF_CUDA(cudaFuncGetAttributes(&a, kernel));
                WGF_CHECK(a.numRegs >= kStartRegs, WGF_ERR_CUDA, "the 4-bit product was built with fewer registers than it shares out");
                WGF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom + 1024));
                if (dev.ordinal < 64) done[which] |= 1ull << dev.ordinal;
            }
        }
        dev.begin_launch("q4_tc");
        if (!dev.dry) kernel<<<grid, kThreadsTc, smem, dev.stream>>>(map, p);
        dev.end_launch();
    };
    if (parts > 1) go(q4_tc_kernel<__nv_bfloat16, 3>, 0);
    else if (dtype == DType::BF16) go(q4_tc_kernel<__nv_bfloat16, 1>, 1);
    else go(q4_tc_kernel<__half, 1>, 2);
}

}  // namespace wgf
