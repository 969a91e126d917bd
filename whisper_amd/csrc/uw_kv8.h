// The 8-bit paged key/value cache: layout, code conversions and the bookkeeping shared by its kernels.
//
// A page ("block") holds P tokens (16 .. 256, a power of two) of every kv head.  Per head: K codes row by row [P][D], V codes
// transposed [D][P].  Both are then read along the index the attention product sums over -- D for q.k, the tokens for p.v -- as
// 16-byte chunks that are MFMA operands as they lie, with no transpose between memory and register.  One f32 scale per page, head
// and half; value = code * scale.  Two code formats, both exact in bf16 (8 significant bits):
//   int8  codes -127 .. 127, scale = largest |x| / 127
//   e4m3  (1-4-3, no infinities, largest 448), scale = the smallest power of two that fits
#pragma once
#include "../../include/uw_hip.h"
#include "uw_common.h"

struct Kv8View {
    uint8_t *k, *v;          // [n_pages][Hkv][P][D], [n_pages][Hkv][D][P]
    float *ks, *vs;          // [n_pages][Hkv]
    int n_pages, Hkv, P, log2P, D;
    const int32_t* table;    // [B][width] page of each block of a sequence
    int width;
};

// New tokens (or query tokens) of B sequences: T each in [B][T] order, or packed one behind the other with tok_start [B + 1].
struct TokSpan {
    const int32_t* tok_start;   // null: uniform
    int B, T;                   // T: tokens per sequence (uniform only)
    long N;                     // rows altogether
    __device__ __forceinline__ long first(int b) const { return tok_start ? (long)tok_start[b] : (long)b * T; }
    // tokens of sequence b; a malformed tok_start gives 0 rather than rows outside [0, N)
    __device__ __forceinline__ int count(int b) const
    {
        if (!tok_start) return T;
        const long s = tok_start[b], e = tok_start[b + 1];
        return (s < 0 || e > N || e < s) ? 0 : (int)(e - s);
    }
};

// page of block `blk` of sequence b, or -1 (outside the table, or an id outside the cache)
__device__ __forceinline__ int kv8_page(const Kv8View& c, int b, long blk)
{
    if (blk < 0 || blk >= c.width) return -1;
    const int id = c.table[(long)b * c.width + blk];
    return (id < 0 || id >= c.n_pages) ? -1 : id;
}

// ---- code <-> value ---------------------------------------------------------------------------------
template <int F> __device__ __forceinline__ float kv8_decode(uint8_t c);
template <> __device__ __forceinline__ float kv8_decode<UW_KV8_INT8>(uint8_t c) { return (float)(int8_t)c; }
template <> __device__ __forceinline__ float kv8_decode<UW_KV8_E4M3>(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

// Codes of four values under the reciprocal scale r.  int8: the 48-bit product is taken in f64, so that it is rounded once and the
// code is the definition's whatever the order of evaluation; e4m3: r is a power of two, the f32 product is exact where it matters.
template <int F> __device__ __forceinline__ unsigned kv8_encode4(const float* x, float r);
template <> __device__ __forceinline__ unsigned kv8_encode4<UW_KV8_INT8>(const float* x, float r)
{
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = (int)rint((double)x[i] * (double)r);       // |product| < 128: r fits the block's largest value
        w |= ((unsigned)max(-127, min(127, q)) & 255u) << (8 * i);
    }
    return w;
}
template <> __device__ __forceinline__ unsigned kv8_encode4<UW_KV8_E4M3>(const float* x, float r)
{
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(x[i] * r, -448.f), 448.f);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
}

// smallest e with 2^e >= v, v a positive normal number
__device__ __forceinline__ int ceil_log2(double v)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(v);
    return (int)((u >> 52) & 0x7ff) - 1023 + ((u & 0xfffffffffffffull) ? 1 : 0);
}
// scale of a block that begins with values up to amax (0: a block of zeros)
template <int F> __device__ __forceinline__ float kv8_base_scale(float amax)
{
    if (!(amax > 0.f)) return 0.f;
    if (F == UW_KV8_INT8) return fmaxf(amax / 127.0f, 0x1p-126f);
    return __uint_as_float((unsigned)(max(ceil_log2((double)amax / 448.0), -126) + 127) << 23);
}
// powers of two by which the scale s > 0 of a block with tokens in it has to grow for values up to amax (0: it fits).  Growing by
// powers of two bounds what repeated re-rounding of the old codes can add up to (int8: one step in all, e4m3: nothing but
// underflow); a block that followed its largest value exactly would re-round at every new maximum.
template <int F> __device__ __forceinline__ int kv8_growth(float amax, float s)
{
    const double need = (double)amax / ((F == UW_KV8_INT8 ? 127.5 : 448.0) * (double)s);   // int8: 127.5 still rounds to within half a step of 127
    return need > 1.0 ? ceil_log2(need) : 0;
}
