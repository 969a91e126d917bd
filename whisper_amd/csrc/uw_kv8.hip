// The 8-bit paged key/value cache: append and read back.
#include "../../include/uw_hip.h"
#include "uw_kv8.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

// blocks that n tokens from position pos on touch (positions before the first lie in blocks before the first, which have no page)
__device__ __forceinline__ int touched(int pos, int n, int log2P)
{
    return n <= 0 ? 0 : (int)(((unsigned)(pos & ((1 << log2P) - 1)) + (unsigned)n - 1) >> log2P) + 1;
}

// ------------------------------------------------------------------------------------------------
// Append and read: a workgroup per touched block, head and half, TPB threads (64 for a few tokens, so that a decode step's tokens do
// not each hold four waves).  Both are bound by memory: values once, codes once, nothing between.  V passes through LDS on its way to
// or from [D][P], a channel's tokens at a pitch of P + 4 bytes, so that the words of a wave fall into different banks.
// Measured, calls back to back in a graph: 32 x 1500 tokens of 12 heads of 64, bf16 (221 MB each way) stored in 51.5 us, 4.3 TB/s, read back in
// 42.4, 5.2 TB/s (a large copy: 4.65); the newest token of 128 sequences stored in 6.7 us, which is one chain of length, page, value and
// scale, not bandwidth (0.6 MB).

struct Block {           // one block of a call
    int b, r0, rows;            // sequence, first row in the block, rows of the call
    long blk;                   // which block of the sequence
    long row;                   // their first row of the call, as an element offset into the token array (without the head)
};

__device__ __forceinline__ bool find_block(const Kv8View& c, const TokSpan& ts, const TokArg& a, const int32_t* pos_of, Block& o)
{
    int j;
    const int item = blockIdx.x / c.Hkv;       // heads run fastest: neighbours in the token array are at work at the same time
    if (ts.tok_start) {
        if (!locate(item, ts.B, [&](int i) { return touched(pos_of[i], ts.count(i), c.log2P); }, o.b, j)) return false;
    } else {
        const int per = (ts.T + c.P - 2) / c.P + 1;
        o.b = item / per;
        j = item % per;
        if (j >= touched(pos_of[o.b], ts.T, c.log2P)) return false;
    }
    const int pos = pos_of[o.b], n = ts.count(o.b);
    const int in = pos & (c.P - 1), t0 = max(0, (j << c.log2P) - in);      // place in its block of the first token; the call's first token in block j
    o.blk = (long)(pos >> c.log2P) + j;
    o.r0 = j ? 0 : in;
    o.rows = min(n - t0, c.P - o.r0);
    o.row = ts.tok_start ? (ts.first(o.b) + t0) * a.sT : (long)o.b * a.sB + (long)t0 * a.sT;
    return true;
}

// Units of work.  K: a piece of 8 channels of a token (8 bytes of codes).  V: 8 channels of 4 tokens (a token group, aligned in the
// block; 4 channels when read), transposed in registers -- its codes are 4 bytes of each channel.
// (the new tokens are read once: their lines need not stay)
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
template <typename T, int N> __device__ __forceinline__ void load_n(const void* p, long at, float* x)
{
    static_assert(N == 8, "16 bytes of bf16");
    if constexpr (sizeof(T) == 2) {
        unsigned w[N / 2];
        const u32x4 v = __builtin_nontemporal_load((const u32x4*)((const T*)p + at));
        w[0] = v[0]; w[1] = v[1]; w[2] = v[2]; w[3] = v[3];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) { x[2 * i] = bf16lo(w[i]); x[2 * i + 1] = bf16hi(w[i]); }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 v = __builtin_nontemporal_load((const f32x4*)((const T*)p + at + i));
            x[i] = v[0]; x[i + 1] = v[1]; x[i + 2] = v[2]; x[i + 3] = v[3];
        }
    }
}
template <typename T, int N> __device__ __forceinline__ void store_n(void* p, long at, const float* x)
{
    if constexpr (sizeof(T) == 2) {
        typedef __bf16 V __attribute__((ext_vector_type(N)));
        V v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (bf16_t)x[i];
        *(V*)((T*)p + at) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) *(f32x4*)((T*)p + at + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    }
}

// largest |x| by its bits, which order like the values, with infinity and NaN above every number
template <int N> __device__ __forceinline__ unsigned largest(unsigned mx, const float* x)
{
#pragma unroll
    for (int i = 0; i < N; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7fffffffu);
    return mx;
}

// scale of a block whose new values reach up to amax (its bits mx), r0 earlier tokens in it; `grow`: powers of two that it grew by
template <int F> __device__ __forceinline__ float next_scale(unsigned mx, int r0, float old_s, int& grow)
{
    const float amax = __uint_as_float(mx);
    grow = 0;
    if (mx >= 0x7f800000u || (r0 > 0 && !(fabsf(old_s) < INFINITY))) return __uint_as_float(0x7fc00000u);
    if (r0 == 0 || old_s <= 0.f) return kv8_base_scale<F>(amax);
    grow = kv8_growth<F>(amax, old_s);
    return ldexpf(old_s, grow);
}

// `words` words of each of `lines` lines of codes `pitch` bytes apart, re-rounded under a scale 2^grow times as large; of a line only the
// first `used` bytes are earlier tokens' codes
template <int F, int TPB> __device__ __forceinline__ void requantise(uint8_t* codes, int lines, int pitch, int used, int grow)
{
    const float down = ldexpf(1.f, -grow);
    const int words = (used + 3) / 4;
    for (int e = threadIdx.x; e < words * lines; e += TPB) {
        unsigned* at = (unsigned*)(codes + (e / words) * pitch + (e % words) * 4);
        const unsigned w = *at;
        float x[4];
        kv8_decode4<F>(w, x);
        const int keep = min(4, used - (e % words) * 4);
        const unsigned m = keep == 4 ? ~0u : (1u << (8 * keep)) - 1u;
        *at = (kv8_encode4<F>(x, down) & m) | (w & ~m);
    }
    __syncthreads();
}

template <int F, typename T, int D, int TPB>
__global__ __launch_bounds__(TPB) void kv8_append_kernel(Kv8View c, TokSpan ts, TokArg ka, TokArg va, const int32_t* pos_of)
{
    __shared__ unsigned s_max[TPB / 64];
    extern __shared__ __attribute__((aligned(16))) uint8_t tile[];      // V: [D][P + 4]
    const bool is_v = blockIdx.y;
    const TokArg a = is_v ? va : ka;
    Block k;
    if (!find_block(c, ts, a, pos_of, k)) return;
    const int h = blockIdx.x % c.Hkv, tid = threadIdx.x, P = c.P;
    const long src = k.row + (long)h * a.sH;
    auto block_max = [&](unsigned mx) {
        mx = across_wave(mx, [](unsigned p, unsigned q) { return max(p, q); });
        if constexpr (TPB > 64) {
            if ((tid & 63) == 0) s_max[tid >> 6] = mx;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < TPB / 64; ++w) mx = max(mx, s_max[w]);
        }
        return mx;
    };
    if (!is_v) {
        constexpr int PIECES = D / 8, HELD = 4;       // pieces of a token; pieces a thread keeps between finding the maximum and encoding
        const int n = k.rows * PIECES;
        auto load = [&](int e, float* x) { load_n<T, 8>(a.data, src + (long)(e / PIECES) * a.sT + (e % PIECES) * 8, x); };
        float held[HELD][8];
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
#pragma unroll
            for (int i = 0; i < 8; ++i) held[u][i] = 0.f;
            if (tid + u * TPB < n) load(tid + u * TPB, held[u]);
        }
        // (the page is looked up while the values are on their way)
        const int page = kv8_page(c, k.b, k.blk);
        if (page < 0) return;
        uint8_t* codes = c.k + ((long)page * c.Hkv + h) * P * D;
        float* scale = c.ks + (long)page * c.Hkv + h;
        const float old_s = *scale;
        unsigned mx = 0;
#pragma unroll
        for (int u = 0; u < HELD; ++u) mx = largest<8>(mx, held[u]);
        for (int e = tid + HELD * TPB; e < n; e += TPB) {
            float x[8];
            load(e, x);
            mx = largest<8>(mx, x);
        }
        int grow;
        const float s = next_scale<F>(block_max(mx), k.r0, old_s, grow), rs = s > 0.f ? 1.0f / s : 0.f;
        if (grow) requantise<F, TPB>(codes, 1, 0, k.r0 * D, grow);
        if (tid == 0) *scale = s;
        auto put = [&](int e, const float* x) {
            *(uint2*)(codes + (k.r0 + e / PIECES) * D + (e % PIECES) * 8) = make_uint2(kv8_encode4<F>(x, rs), kv8_encode4<F>(x + 4, rs));
        };
#pragma unroll
        for (int u = 0; u < HELD; ++u)
            if (tid + u * TPB < n) put(tid + u * TPB, held[u]);
        for (int e = tid + HELD * TPB; e < n; e += TPB) {
            float x[8];
            load(e, x);
            put(e, x);
        }
        return;
    }
    constexpr int UNITS = D / 8;
    const int w0 = k.r0 >> 2, words = ((k.r0 + k.rows + 3) >> 2) - w0, n = words * UNITS;      // token groups that hold new tokens
    auto load = [&](int e, float (*x)[8]) {
        const int r = (w0 + e / UNITS) * 4 - k.r0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
            if (r + i >= 0 && r + i < k.rows) load_n<T, 8>(a.data, src + (long)(r + i) * a.sT + (e % UNITS) * 8, x[i]);
        }
    };
    float held[4][8] = {};                              // the unit a thread keeps
    if (tid < n) load(tid, held);
    const int page = kv8_page(c, k.b, k.blk);
    if (page < 0) return;
    uint8_t* codes = c.v + ((long)page * c.Hkv + h) * P * D;
    float* scale = c.vs + (long)page * c.Hkv + h;
    const float old_s = *scale;
    unsigned mx = largest<32>(0, held[0]);
    for (int e = tid + TPB; e < n; e += TPB) {
        float x[4][8];
        load(e, x);
        mx = largest<32>(mx, x[0]);
    }
    int grow;
    const float s = next_scale<F>(block_max(mx), k.r0, old_s, grow), rs = s > 0.f ? 1.0f / s : 0.f;
    if (grow) requantise<F, TPB>(codes, D, P, k.r0, grow);
    if (tid == 0) *scale = s;
    auto put = [&](int e, float (*x)[8]) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = kv8_encode4<F>(x[i] + 4 * q, rs);
            transpose4(w);
#pragma unroll
            for (int j = 0; j < 4; ++j) *(unsigned*)(tile + ((e % UNITS) * 8 + 4 * q + j) * (P + 4) + (w0 + e / UNITS) * 4) = w[j];
        }
    };
    if (tid < n) put(tid, held);
    for (int e = tid + TPB; e < n; e += TPB) {
        float x[4][8];
        load(e, x);
        put(e, x);
    }
    __syncthreads();
    if (k.rows == P) {                                  // a whole block: 16 bytes at a time
        const int per = P / 16;
        for (int e = tid; e < per * D; e += TPB) {
            const unsigned* from = (const unsigned*)(tile + (e / per) * (P + 4) + (e % per) * 16);
            *(uint4*)(codes + e * 16) = make_uint4(from[0], from[1], from[2], from[3]);
        }
        return;
    }
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
    extern __shared__ __attribute__((aligned(16))) uint8_t tile[];
    const bool is_v = blockIdx.y;
    const TokArg a = is_v ? va : ka;
    Block k;
    if (!find_block(c, ts, a, first_of, k)) return;
    const int h = blockIdx.x % c.Hkv, tid = threadIdx.x, P = c.P;
    const long dst = k.row + (long)h * a.sH;
    const int page = kv8_page(c, k.b, k.blk);
    const long at = (long)max(page, 0) * c.Hkv + h;
    const uint8_t* codes = (is_v ? c.v : c.k) + at * P * D;
    const float s = page < 0 ? __uint_as_float(0x7fc00000u) : (is_v ? c.vs : c.ks)[at];
    if (!is_v) {
        constexpr int PIECES = D / 8;
        for (int e = tid; e < k.rows * PIECES; e += TPB) {
            const uint2 w = *(const uint2*)(codes + (k.r0 + e / PIECES) * D + (e % PIECES) * 8);
            float x[8];
            kv8_decode4<F>(w.x, x);
            kv8_decode4<F>(w.y, x + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= s;
            store_n<T, 8>(a.data, dst + (long)(e / PIECES) * a.sT + (e % PIECES) * 8, x);
        }
        return;
    }
    const int g0 = k.r0 >> 4, per = ((k.r0 + k.rows + 15) >> 4) - g0;          // 16-token groups of a channel that are wanted
    for (int e = tid; e < per * D; e += TPB) {
        const int d = e / per, r = (g0 + e % per) * 16;
        const uint4 w = *(const uint4*)(codes + d * P + r);
        unsigned* to = (unsigned*)(tile + d * (P + 4) + r);
        to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
    }
    __syncthreads();
    constexpr int UNITS = D / 4;
    const int w0 = k.r0 >> 2, words = ((k.r0 + k.rows + 3) >> 2) - w0;
    for (int e = tid; e < words * UNITS; e += TPB) {
        const int d = (e % UNITS) * 4, r = (w0 + e / UNITS) * 4;
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *(const unsigned*)(tile + (d + j) * (P + 4) + r);
        transpose4(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r + i < k.r0 || r + i >= k.r0 + k.rows) continue;
            float x[4];
            kv8_decode4<F>(w[i], x);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] *= s;
            store_n<T, 4>(a.data, dst + (long)(r + i - k.r0) * a.sT + d, x);
        }
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
    UW_REQUIRE(touched_bound(&a->seqs, a->cache.page) * a->cache.n_kv_heads < (1 << 24), "%s: too many rows", fn);
    return UW_OK;
}

// One wave per block and head for a decode step's tokens, two otherwise: most of a workgroup's life is waiting for its lengths, its
// page and its values, so many small ones beat few large ones.  One wave / two, back to back in a graph: 128 sequences' newest token stored 6.7 /
// 7.6 us, their last blocks read back 9.4 / 9.8; 32 x 1500 tokens stored 55.7 / 51.5, read back 43.2 / 42.4; 16 x up to 701 f32 tokens of 128
// channels stored 22.1 / 17.4.
bool few_tokens(const uw_kv8_store_args* a)
{
    const long per = a->seqs.tok_start ? ceil_div(a->seqs.n_tok, a->seqs.B) : a->seqs.T;
    return per * a->cache.head_dim <= 512;
}

#define KV8_STORE_LAUNCH(NAME, KERNEL)                                                                                              \
    template <int F, typename T, int D> int NAME(const uw_kv8_store_args* a, hipStream_t s)                                         \
    {                                                                                                                               \
        const Kv8View c = view_of(&a->cache, &a->seqs);                                                                             \
        const dim3 grid((unsigned)(touched_bound(&a->seqs, c.P) * c.Hkv), 2);                                                          \
        const size_t lds = (size_t)D * (c.P + 4);                                                                                   \
        const TokSpan ts = span_of(&a->seqs);                                                                                       \
        if (few_tokens(a)) hipLaunchKernelGGL((KERNEL<F, T, D, 64>), grid, dim3(64), lds, s, c, ts, arg_of(&a->k), arg_of(&a->v), a->seqs.len); \
        else hipLaunchKernelGGL((KERNEL<F, T, D, 128>), grid, dim3(128), lds, s, c, ts, arg_of(&a->k), arg_of(&a->v), a->seqs.len); \
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
