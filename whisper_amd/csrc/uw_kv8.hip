// The 8-bit paged key/value cache: append and read back.
#include "../../include/uw_hip.h"
#include "uw_kv8.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

// blocks that n tokens from position pos on touch
__device__ __forceinline__ int touched(int pos, int n, int log2P)
{
    return (n <= 0 || pos < 0) ? 0 : (int)((((long)pos + n - 1) >> log2P) - (pos >> log2P) + 1);
}

// ------------------------------------------------------------------------------------------------
// Append and read: a workgroup per touched block, head and half, TPB threads (64 for a few tokens, so that a decode step's tokens do
// not each hold four waves).  Tokens move in pieces of 8 values, 16 bytes of bf16; V passes through LDS to be transposed, where a
// channel's tokens have a pitch of P + 4 bytes: the 8 bytes of a piece then fall into 8 banks.

struct Block {           // one block of a call
    int b, page, r0, rows;      // sequence, page (-1: none), first row in the block, rows of the call
    long row;                   // their first row of the call, as an element offset into the token array (without the head)
};

__device__ __forceinline__ bool find_block(const Kv8View& c, const TokSpan& ts, const TokArg& a, const int32_t* pos_of, Block& o)
{
    int j;
    if (ts.tok_start) {
        if (!locate(blockIdx.x, ts.B, [&](int i) { return touched(pos_of[i], ts.count(i), c.log2P); }, o.b, j)) return false;
    } else {
        const int per = (ts.T + c.P - 2) / c.P + 1;
        o.b = blockIdx.x / per;
        j = blockIdx.x % per;
        if (j >= touched(pos_of[o.b], ts.T, c.log2P)) return false;
    }
    const int pos = pos_of[o.b], n = ts.count(o.b);
    const long blk = (pos >> c.log2P) + j, p0 = blk << c.log2P;      // first position of the block
    const int t0 = (int)max(0l, p0 - pos), t1 = (int)min((long)n, p0 + c.P - pos);
    o.page = kv8_page(c, o.b, blk);
    o.r0 = (int)(pos + t0 - p0);
    o.rows = t1 - t0;
    o.row = ts.tok_start ? (ts.first(o.b) + t0) * a.sT : (long)o.b * a.sB + (long)t0 * a.sT;
    return true;
}

// 8 values of a token, 16-byte aligned
template <typename T> __device__ __forceinline__ void load8(const void* p, long at, float* x);
template <> __device__ __forceinline__ void load8<bf16_t>(const void* p, long at, float* x)
{
    const uint4 w = *(const uint4*)((const bf16_t*)p + at);
    x[0] = bf16lo(w.x); x[1] = bf16hi(w.x); x[2] = bf16lo(w.y); x[3] = bf16hi(w.y);
    x[4] = bf16lo(w.z); x[5] = bf16hi(w.z); x[6] = bf16lo(w.w); x[7] = bf16hi(w.w);
}
template <> __device__ __forceinline__ void load8<float>(const void* p, long at, float* x)
{
    const f32x4 a = *(const f32x4*)((const float*)p + at), b = *(const f32x4*)((const float*)p + at + 4);
    x[0] = a[0]; x[1] = a[1]; x[2] = a[2]; x[3] = a[3]; x[4] = b[0]; x[5] = b[1]; x[6] = b[2]; x[7] = b[3];
}
template <typename T> __device__ __forceinline__ void store8(void* p, long at, const float* x);
template <> __device__ __forceinline__ void store8<bf16_t>(void* p, long at, const float* x)
{
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16_t)x[i];
    *(uint4*)((bf16_t*)p + at) = __builtin_bit_cast(uint4, v);
}
template <> __device__ __forceinline__ void store8<float>(void* p, long at, const float* x)
{
    *(f32x4*)((float*)p + at) = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)((float*)p + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
}

// four codes of a word, re-rounded under a scale 2^grow times as large (`down` = 2^-grow)
template <int F> __device__ __forceinline__ unsigned requantise4(unsigned w, float down)
{
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = kv8_decode<F>((uint8_t)(w >> (8 * i)));
    return kv8_encode4<F>(x, down);
}

template <int F, typename T, int D, int TPB>
__global__ __launch_bounds__(TPB) void kv8_append_kernel(Kv8View c, TokSpan ts, TokArg ka, TokArg va, const int32_t* pos_of)
{
    constexpr int PIECES = D / 8, HELD = 4;           // pieces per token; pieces a thread keeps between the two passes
    __shared__ unsigned s_max[TPB / 64];
    extern __shared__ __attribute__((aligned(16))) uint8_t tile[];      // V: [D][P + 4]
    const bool is_v = blockIdx.z;
    const TokArg a = is_v ? va : ka;
    Block k;
    if (!find_block(c, ts, a, pos_of, k) || k.page < 0) return;
    const int h = blockIdx.y, tid = threadIdx.x, P = c.P;
    const long src = k.row + (long)h * a.sH;
    uint8_t* codes = (is_v ? c.v : c.k) + ((long)k.page * c.Hkv + h) * P * D;
    float* scale = (is_v ? c.vs : c.ks) + (long)k.page * c.Hkv + h;
    const float old_s = *scale;
    const int n = k.rows * PIECES;

    // largest |x| by its bits: they order like the values, with infinity and NaN above every number
    float held[HELD][8];
    unsigned mx = 0;
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
        const int e = tid + u * TPB;
        if (e < n) load8<T>(a.data, src + (long)(e / PIECES) * a.sT + (e % PIECES) * 8, held[u]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) held[u][i] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < HELD; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(held[u][i]) & 0x7fffffffu);
    for (int e = tid + HELD * TPB; e < n; e += TPB) {
        float x[8];
        load8<T>(a.data, src + (long)(e / PIECES) * a.sT + (e % PIECES) * 8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
    if constexpr (TPB > 64) {
        if ((tid & 63) == 0) s_max[tid >> 6] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TPB / 64; ++w) mx = max(mx, s_max[w]);
    }
    const float amax = __uint_as_float(mx);
    float s;
    int grow = 0;
    if (mx >= 0x7f800000u || (k.r0 > 0 && !(fabsf(old_s) < INFINITY))) {
        s = __uint_as_float(0x7fc00000u);
    } else if (k.r0 == 0 || old_s <= 0.f) {
        s = kv8_base_scale<F>(amax);
    } else {
        grow = kv8_growth<F>(amax, old_s);
        s = ldexpf(old_s, grow);
    }
    if (grow) {          // the earlier tokens' codes, a word at a time; what lies behind them in a word is written over below
        const float down = ldexpf(1.f, -grow);
        const int words = is_v ? (k.r0 + 3) / 4 : k.r0 * D / 4, lines = is_v ? D : 1;
        for (int e = tid; e < words * lines; e += TPB) {
            unsigned* at = (unsigned*)(codes + (is_v ? (e / words) * P + (e % words) * 4 : e * 4));
            const unsigned w = *at;
            const int keep = is_v ? min(4, k.r0 - (e % words) * 4) : 4;        // bytes that are earlier tokens
            const unsigned m = keep == 4 ? ~0u : (1u << (8 * keep)) - 1u;
            *at = (requantise4<F>(w, down) & m) | (w & ~m);
        }
        __syncthreads();
    }
    if (tid == 0) *scale = s;
    const float rs = s > 0.f ? 1.0f / s : 0.f;
    auto put = [&](int e, const float* x) {
        const int r = e / PIECES, d = (e % PIECES) * 8;
        const unsigned lo = kv8_encode4<F>(x, rs), hi = kv8_encode4<F>(x + 4, rs);
        if (!is_v) {
            *(uint2*)(codes + (k.r0 + r) * D + d) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                tile[(d + i) * (P + 4) + k.r0 + r] = (uint8_t)(lo >> (8 * i));
                tile[(d + 4 + i) * (P + 4) + k.r0 + r] = (uint8_t)(hi >> (8 * i));
            }
        }
    };
#pragma unroll
    for (int u = 0; u < HELD; ++u)
        if (tid + u * TPB < n) put(tid + u * TPB, held[u]);
    for (int e = tid + HELD * TPB; e < n; e += TPB) {
        float x[8];
        load8<T>(a.data, src + (long)(e / PIECES) * a.sT + (e % PIECES) * 8, x);
        put(e, x);
    }
    if (!is_v) return;
    __syncthreads();
    const int w0 = k.r0 >> 2, words = ((k.r0 + k.rows + 3) >> 2) - w0;         // words of a channel that hold new tokens
    for (int e = tid; e < words * D; e += TPB) {
        const int d = e / words, r = (w0 + e % words) * 4;
        const uint8_t* from = tile + d * (P + 4) + r;
        uint8_t* to = codes + d * P + r;
        if (r >= k.r0 && r + 4 <= k.r0 + k.rows) {
            *(unsigned*)to = *(const unsigned*)from;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r + i >= k.r0 && r + i < k.r0 + k.rows) to[i] = from[i];
        }
    }
}

template <int F, typename T, int D, int TPB>
__global__ __launch_bounds__(TPB) void kv8_read_kernel(Kv8View c, TokSpan ts, TokArg ka, TokArg va, const int32_t* first_of)
{
    constexpr int PIECES = D / 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t tile[];
    const bool is_v = blockIdx.z;
    const TokArg a = is_v ? va : ka;
    Block k;
    if (!find_block(c, ts, a, first_of, k)) return;
    const int h = blockIdx.y, tid = threadIdx.x, P = c.P;
    const long dst = k.row + (long)h * a.sH;
    const long at = (long)max(k.page, 0) * c.Hkv + h;
    const uint8_t* codes = (is_v ? c.v : c.k) + at * P * D;
    const float s = k.page < 0 ? __uint_as_float(0x7fc00000u) : (is_v ? c.vs : c.ks)[at];
    if (is_v) {
        const int w0 = k.r0 >> 2, words = ((k.r0 + k.rows + 3) >> 2) - w0;
        for (int e = tid; e < words * D; e += TPB) {
            const int d = e / words, r = (w0 + e % words) * 4;
            *(unsigned*)(tile + d * (P + 4) + r) = *(const unsigned*)(codes + d * P + r);
        }
        __syncthreads();
    }
    for (int e = tid; e < k.rows * PIECES; e += TPB) {
        const int r = e / PIECES, d = (e % PIECES) * 8;
        uint2 w;
        if (!is_v) {
            w = *(const uint2*)(codes + (k.r0 + r) * D + d);
        } else {
            w = make_uint2(0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w.x |= (unsigned)tile[(d + i) * (P + 4) + k.r0 + r] << (8 * i);
                w.y |= (unsigned)tile[(d + 4 + i) * (P + 4) + k.r0 + r] << (8 * i);
            }
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = kv8_decode<F>((uint8_t)(w.x >> (8 * i))) * s;
            x[4 + i] = kv8_decode<F>((uint8_t)(w.y >> (8 * i))) * s;
        }
        store8<T>(a.data, dst + (long)r * a.sT + d, x);
    }
}

// ---- host side --------------------------------------------------------------------------------------
// upper bound of the blocks a call touches, known without reading the lengths: n tokens touch at most (n - 1) / P + 2
long touched_bound(const uw_kv8_seqs* t, int P)
{
    if (t->tok_start) return t->n_tok / P + 2l * std::min((long)t->B, (long)t->n_tok);
    return (long)t->B * ((t->T + P - 2) / P + 1);
}

int check_store(const char* fn, const uw_kv8_store_args* a)
{
    UW_REQUIRE(a, "%s: null arguments", fn);
    RUN(check_cache(fn, &a->cache));
    RUN(check_seqs(fn, &a->seqs));
    RUN(check_tokens(fn, "k", &a->k, &a->seqs));
    RUN(check_tokens(fn, "v", &a->v, &a->seqs));
    UW_REQUIRE(touched_bound(&a->seqs, a->cache.page) < (1 << 24), "%s: too many rows", fn);
    return UW_OK;
}

// one wave per block and head while that leaves each lane at most one piece of 8 values (a decode step's tokens), else four
bool few_tokens(const uw_kv8_store_args* a)
{
    const long per = a->seqs.tok_start ? ceil_div(a->seqs.n_tok, a->seqs.B) : a->seqs.T;
    return per * a->cache.head_dim <= 512;
}

#define KV8_STORE_LAUNCH(NAME, KERNEL)                                                                                              \
    template <int F, typename T, int D> int NAME(const uw_kv8_store_args* a, hipStream_t s)                                         \
    {                                                                                                                               \
        const Kv8View c = view_of(&a->cache, &a->seqs);                                                                             \
        const dim3 grid((unsigned)touched_bound(&a->seqs, c.P), c.Hkv, 2);                                                          \
        const size_t lds = (size_t)D * (c.P + 4);                                                                                   \
        const TokSpan ts = span_of(&a->seqs);                                                                                       \
        if (few_tokens(a)) hipLaunchKernelGGL((KERNEL<F, T, D, 64>), grid, dim3(64), lds, s, c, ts, arg_of(&a->k), arg_of(&a->v), a->seqs.len); \
        else hipLaunchKernelGGL((KERNEL<F, T, D, 256>), grid, dim3(256), lds, s, c, ts, arg_of(&a->k), arg_of(&a->v), a->seqs.len); \
        UW_LAUNCH_CHECK();                                                                                                          \
        return UW_OK;                                                                                                               \
    }
KV8_STORE_LAUNCH(launch_append, kv8_append_kernel)
KV8_STORE_LAUNCH(launch_read, kv8_read_kernel)

}  // namespace

extern "C" {

int uw_kv8_append(const uw_kv8_store_args* a, void* stream)
{
    RUN(check_store("uw_kv8_append", a));
    if (a->seqs.n_tok == 0) return UW_OK;
#define CALL(F, T) RUN((a->cache.head_dim == 64 ? launch_append<F, T, 64>(a, (hipStream_t)stream) : launch_append<F, T, 128>(a, (hipStream_t)stream)))
    KV8_DISPATCH(a->cache.format, a->seqs.dtype, CALL);
#undef CALL
    return UW_OK;
}

int uw_kv8_read(const uw_kv8_store_args* a, void* stream)
{
    RUN(check_store("uw_kv8_read", a));
    if (a->seqs.n_tok == 0) return UW_OK;
#define CALL(F, T) RUN((a->cache.head_dim == 64 ? launch_read<F, T, 64>(a, (hipStream_t)stream) : launch_read<F, T, 128>(a, (hipStream_t)stream)))
    KV8_DISPATCH(a->cache.format, a->seqs.dtype, CALL);
#undef CALL
    return UW_OK;
}

}  // extern "C"
