// Device-side view of the paged key-value cache shared by the append and attention kernels.
//
// A layer's pool is [n_pages][Hkv][page_size][D] of 16-bit values: a (page, kv head) is one contiguous
// run of page_size rows, so an attention kernel, which works on one kv head, reads whole runs.
// The tables, lengths and token offsets are device data the host never sees; every page id and
// position is checked where it is used (kDevBadPage / kDevBadToken in the status word, and the
// access is replaced by one in bounds or left out).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "moe_common.cuh"
#include "moe_internal.h"

namespace moe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Round to nearest even, as every store of this cache and of attention outputs does.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 2^x (the hardware's approximation, within 2 ulp; 2^-inf = 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 values as a pair of 16-bit ones (x low), and the pair of what that rounding left over: the
// two pieces together hold a value to twice the type's precision.
template <typename C> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename C> __device__ __forceinline__ uint32_t pack_rest(uint32_t packed, float x, float y);
template <> __device__ __forceinline__ uint32_t pack_rest<__half>(uint32_t packed, float x, float y) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack2<__half>(x - v.x, y - v.y);
}
template <> __device__ __forceinline__ uint32_t pack_rest<__nv_bfloat16>(uint32_t packed, float x, float y) {
    return pack2<__nv_bfloat16>(x - __uint_as_float(packed << 16), y - __uint_as_float(packed & 0xFFFF0000u));
}

// Four output values v * inv, rounded to the output's type.
__device__ __forceinline__ void store4(float* out, float4 v, float inv) {
    *reinterpret_cast<float4*>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}
template <typename C> __device__ __forceinline__ void store4(C* out, float4 v, float inv) {
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<C>(v.x * inv, v.y * inv), pack2<C>(v.z * inv, v.w * inv));
}

// The exponent e that takes a query row of largest magnitude mx to [2^14, 2^15) in f16 pieces (as far as
// a normal f32 power goes; 0 for an all-zero or not finite row), and 2^e, exact.
__device__ __forceinline__ int row_exponent(float mx) {
    return mx > 0.f && mx < INFINITY ? min(126, 141 - (__float_as_int(mx) >> 23)) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The page of table entry p, or page 0 and an error for an id outside the cache.
__device__ __forceinline__ uint32_t checked_page(int p, uint32_t n_pages, int* status) {
    if (static_cast<uint32_t>(p) < n_pages) return static_cast<uint32_t>(p);
    set_dev_error(status, kDevBadPage);
    return 0;
}

// A sequence's length as the kernels use it: a negative one, or one past its table row, is an
// error and counts as the nearest valid length.
__device__ __forceinline__ int checked_len(int len, const KvBatch& b, int* status) {
    const long long cap = static_cast<long long>(b.max_pages) * b.page_size;
    if (len >= 0 && len <= cap) return len;
    set_dev_error(status, kDevBadToken);
    return len < 0 ? 0 : static_cast<int>(cap);
}

// Whether a sequence can have the packed rows [from, to) of T.
__device__ __forceinline__ bool right_offsets(int from, int to, int T) { return from >= 0 && from <= to && to <= T; }

// The sequence whose packed tokens [cu[s], cu[s+1]) hold token t, or -1 behind the last one (and
// in front of the first); without offsets every sequence has one token.  By a whole warp: 32 offsets at a
// time, so that up to 31 sequences take one round of loads.
__device__ __forceinline__ int warp_seq_of_token(const KvBatch& b, int t, int lane) {
    if (!b.cu) return t < b.n_seqs ? t : -1;
    int lo = 0, hi = b.n_seqs + 1;  // offsets [lo, hi): the last one <= t among them
    if (t < b.cu[0] || t >= b.cu[b.n_seqs]) return -1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const int n = __popc(__ballot_sync(0xffffffffu, i < hi && b.cu[i < hi ? i : lo] <= t));  // offsets ascend: the first n lanes
        if (n == 0) return -1;  // offsets that do not ascend
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return min(lo, b.n_seqs - 1);
}

}  // namespace moe
