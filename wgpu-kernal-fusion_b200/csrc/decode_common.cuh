// Pieces that the kernels of the decode path share: conversions, wide loads, the norm and rotation
// of one head, and the rounding of a value to its code.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace wgf {
namespace decode {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements moved as one access
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

// Shared memory by its own 32-bit addresses
__device__ __forceinline__ unsigned shared_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 shared_16(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float2 shared_float2(unsigned at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned shared_word(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
// From global to shared memory without waiting: 16, 8 or 4 bytes
__device__ __forceinline__ void copy16_at(unsigned dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES> __device__ __forceinline__ void copy_at(unsigned dst, const void* src) {
    static_assert(BYTES == 4 || BYTES == 8, "");
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy16(void* dst, const void* src) { copy16_at(shared_address(dst), src); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// round-half-even(k * x / den) for an integer k <= 127 and den > 0, |k * x / den| <= 127 or so, as if
// the quotient were exact: the codes do not depend on how a division rounds.  k * x is held in two
// floats and the remainder of the nearest integer is exact by the fused multiply-add, so comparing it with
// half a step tells which side of the border the value is on.
__device__ __forceinline__ int exact_code(float x, float k, float den, float inv) {
    const float p = __fmul_rn(k, x), pl = __fmaf_rn(k, x, -p);
    float r = rintf(__fmul_rn(p, inv));
    const float e = __fmaf_rn(-r, den, p);         // p - r * den, exact
    const float h = 0.5f * den;
    const float over = (e - h) + pl, under = (e + h) + pl;   // > 0: above the upper border; < 0: below the lower one
    if (over > 0.f || (over == 0.f && (((int)r) & 1))) r += 1.f;
    else if (under < 0.f || (under == 0.f && (((int)r) & 1))) r -= 1.f;
    return (int)r;
}

// The largest |x| as an ordered integer: NaN above infinity above every number, so that a block that holds
// either is told apart whatever the order of its values.
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// ---- one head: y = x / sqrt(mean(x^2) + eps) * w, then rotated by the position's angle -------------------
// A group of `lanes` (a power of two, at most 32, neighbours in a warp) holds a row: lane l has the chunks
// l, l + lanes, ... of VEC values of the first half, and the same chunks of the second half, which are the
// partners of the rotation.  A row stays as it was loaded until it is used.  Everything is f32 and rounded once.
//
// What a position does to a head: with w the weight,
//   out_lo = (x_lo (w_lo cos) - x_hi (w_hi sin)) r,  out_hi = (x_hi (w_hi cos) + x_lo (w_lo sin)) r,
// so weight and angle are multiplied once for all heads of a token.
template <typename T, int VEC, int NCH> struct Turn {
    float lc[NCH][VEC], ls[NCH][VEC], hc[NCH][VEC], hs[NCH][VEC];
    __device__ __forceinline__ void load(const T* w, const T* cos, const T* sin, int half, int lane, int lanes) {
        typedef Pack<T, VEC> V;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (lane + c * lanes) * VEC, at = j < half ? j : 0;
            const V a = *reinterpret_cast<const V*>(w + at), b = *reinterpret_cast<const V*>(w + half + at);
            const V cs = *reinterpret_cast<const V*>(cos + at), sn = *reinterpret_cast<const V*>(sin + at);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float lo = to_f<T>(a.v[e]), hi = to_f<T>(b.v[e]), x = to_f<T>(cs.v[e]), y = to_f<T>(sn.v[e]);
                lc[c][e] = lo * x;
                ls[c][e] = lo * y;
                hc[c][e] = hi * x;
                hs[c][e] = hi * y;
            }
        }
    }
};
template <typename T, int VEC, int NCH> struct HeadRow {
    Pack<T, VEC> lo[NCH], hi[NCH];

    __device__ __forceinline__ void load(const T* row, int half, int lane, int lanes) {
        typedef Pack<T, VEC> V;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (lane + c * lanes) * VEC;
            if (j < half) {
                lo[c] = *reinterpret_cast<const V*>(row + j);
                hi[c] = *reinterpret_cast<const V*>(row + half + j);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) lo[c].v[e] = hi[c].v[e] = from_f<T>(0.f);
            }
        }
    }
    // All 32 lanes of the warp take part.
    __device__ __forceinline__ float inverse_rms(int half, int lanes, float eps) const {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a = to_f<T>(lo[c].v[e]), b = to_f<T>(hi[c].v[e]);
                s += a * a;
                s += b * b;
            }
        for (int m = lanes >> 1; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        return 1.0f / sqrtf(s / (float)(2 * half) + eps);
    }
    // The normed and rotated row, rounded
    __device__ __forceinline__ HeadRow turned(const Turn<T, VEC, NCH>& t, float r) const {
        HeadRow y;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a = to_f<T>(lo[c].v[e]), b = to_f<T>(hi[c].v[e]);
                y.lo[c].v[e] = from_f<T>((a * t.lc[c][e] - b * t.hs[c][e]) * r);
                y.hi[c].v[e] = from_f<T>((b * t.hc[c][e] + a * t.ls[c][e]) * r);
            }
        return y;
    }
    __device__ __forceinline__ void store(T* row, int half, int lane, int lanes) const {
        typedef Pack<T, VEC> V;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (lane + c * lanes) * VEC;
            if (j >= half) continue;
            *reinterpret_cast<V*>(row + j) = lo[c];
            *reinterpret_cast<V*>(row + half + j) = hi[c];
        }
    }
};

}  // namespace decode
}  // namespace wgf
