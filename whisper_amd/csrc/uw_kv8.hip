// The 8-bit paged key/value cache: append, read back, attention.
#include "../../include/uw_hip.h"
#include "uw_kv8.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

struct TokArg {
    void* data;
    long sB, sT, sH;
};

// The idx-th (sequence, block) pair of a call, blocks counted over the sequences in order; false past the last one.  cnt(b) =
// blocks of sequence b.  Every wave works it out for itself: 64 sequences per step, a shuffle scan each.
template <typename CNT> __device__ __forceinline__ bool locate(long idx, int B, CNT cnt, int& b_out, int& j_out)
{
    const int lane = threadIdx.x & 63;
    long base = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int n = (b0 + lane < B) ? cnt(b0 + lane) : 0;
        long incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long up = __shfl_up(incl, o, 64);
            if (lane >= o) incl += up;
        }
        const unsigned long long over = __ballot(base + incl > idx);
        if (over) {
            const int w = __ffsll((long long)over) - 1;
            b_out = b0 + w;
            j_out = (int)(idx - base - __shfl(incl - n, w, 64));
            return true;
        }
        base += __shfl(incl, 63, 64);
    }
    return false;
}

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

// ------------------------------------------------------------------------------------------------
// Attention.  Rows of one kv head are its G query heads of every query token, token-major: row = t * G + g.  A wave works on 64
// keys at a time and 16 * RT rows, in registers throughout:
//   S^T = K Q^T    16x16x32 MFMA, A = K codes as bf16 (exact), B = Q; lane (row = lane & 15, g = lane >> 4) gets for tile t the keys
//                  16 g + 4 t + 0..3, because row slot r of tile t holds key 16 (r >> 2) + 4 t + (r & 3)
//   O^T = V^T P^T  A = V codes as they lie (16 consecutive keys 16 g .. of one channel), B = P straight from those lanes
// so neither K nor V nor P passes through LDS.  Scales multiply the scores (K) and the probabilities (V) -- one per 16 keys at
// least, so one per lane.  Running maximum, sum and output in f32.  f32 queries and probabilities enter as three bf16 planes (24
// bits): the codes being exact in bf16, that is f32 arithmetic at the bf16 rate.  bf16 queries are exact; their probabilities are
// rounded to bf16 (2^-9 of each, independently), which is what the output is rounded to anyway.
struct AttnArgs {
    Kv8View c;
    TokSpan ts;
    TokArg q, o;
    float* lse;
    const int32_t* kv_len;
    float* part;         // [rows][H][n_split][D + 4] partial results (output, maximum, sum) when n_split > 1
    int H, G, causal, n_split;
    int tiles, groups;   // workgroups per sequence (uniform), and of all sequences
    int lds_rows;        // rows of a tile that can be in use
    float scale2;        // |scale| * log2(e)
    unsigned neg;        // sign bit of scale, moved to the queries
};

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// 8 codes -> an MFMA operand chunk
template <int F> __device__ __forceinline__ bf16x8 codes8(unsigned a, unsigned b);
template <> __device__ __forceinline__ bf16x8 codes8<UW_KV8_E4M3>(unsigned a, unsigned b)
{
    union { bf16x2 p[4]; bf16x8 v; } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return u.v;
}
template <> __device__ __forceinline__ bf16x8 codes8<UW_KV8_INT8>(unsigned a, unsigned b)
{
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (__bf16)(float)(int8_t)(a >> (8 * i));
        v[4 + i] = (__bf16)(float)(int8_t)(b >> (8 * i));
    }
    return v;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// the planes of 8 f32 values
template <int NP> __device__ __forceinline__ void planes(const float* x, bf16x8* out)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float rest = x[e];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const __bf16 part = (__bf16)rest;
            out[n][e] = part;
            rest -= (float)part;
        }
    }
}

// keeps the first n of 16 bytes
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n)
{
    auto m = [&](int k) { return k <= 0 ? 0u : k >= 4 ? ~0u : (1u << (8 * k)) - 1u; };
    return make_uint4(v.x & m(n), v.y & m(n - 4), v.z & m(n - 8), v.w & m(n - 12));
}

// a 16-byte piece of the cache; ONCE: no other workgroup will want it, so it need not stay in L2
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
template <bool ONCE> __device__ __forceinline__ uint4 ld_codes(const void* p)
{
    const u32x4 v = ONCE ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4*)p;
    return make_uint4(v.x, v.y, v.z, v.w);
}

// largest of the four lanes that hold a row (lane & 15 alike), without a trip through LDS; a NaN loses
__device__ __forceinline__ float across_groups_max(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// four channels of a finished row (or of a split's part of it)
template <typename T, int D>
__device__ __forceinline__ void store_row(const AttnArgs& p, int b, long t_first, int kvh, int row, int d, int split, float M, float L, f32x4 acc)
{
    const int t = row / p.G, h = kvh * p.G + row % p.G;
    const long rg = t_first + t;                        // row of the call
    if (p.n_split > 1) {
        float* at = p.part + ((rg * p.H + h) * p.n_split + split) * (D + 4);
        *(f32x4*)(at + d) = acc;
        if (d == 0) { at[D] = M; at[D + 1] = L; }
        return;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    T* out = (T*)p.o.data + (p.ts.tok_start ? rg * p.o.sT : (long)b * p.o.sB + (long)t * p.o.sT) + (long)h * p.o.sH + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = from_f32<T>(acc[k] * inv);
    if (p.lse && d == 0) p.lse[rg * p.H + h] = L == 0.f ? -INFINITY : M * LN2 + logf(L);
}

// WK waves share the keys of a row tile (their results are joined in LDS), WR row tiles per workgroup
template <int F, typename T, int D, int RT, int WK, int WR>
__global__ __launch_bounds__(64 * WK * WR, (RT * D <= 64 && sizeof(T) == 2) ? 4 : RT * D * sizeof(T) <= 512 ? 2 : 1) void kv8_attention_kernel(AttnArgs p)
{
    constexpr int NP = sizeof(T) == 4 ? 3 : 1, ROWS = 16 * RT, HALF = D / 64;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = wave % WK, wr = wave / WK;
    const int rr = lane & 15, g4 = lane >> 4;
    const Kv8View& c = p.c;

    // which sequence, kv head, rows
    // (heads run fastest: the workgroups of a head land on one XCD when their number is a multiple of 8, and share its L2)
    int b, tile;
    const int kvh = blockIdx.x % c.Hkv, rest = blockIdx.x / c.Hkv, split = rest / p.groups, group = rest % p.groups;
    if (p.ts.tok_start) {
        if (!locate(group, p.ts.B, [&](int i) { return (int)(((long)p.ts.count(i) * p.G + ROWS * WR - 1) / (ROWS * WR)); }, b, tile)) return;
    } else {
        b = group / p.tiles;
        tile = group % p.tiles;
    }
    const int n = p.ts.count(b), n_rows = n * p.G;
    if (p.causal) tile = (n_rows + ROWS * WR - 1) / (ROWS * WR) - 1 - tile;      // rows that see most first
    const int row0 = (tile * WR + wr) * ROWS;
    const int len = max(0, p.kv_len[b]);
    const long t_first = p.ts.first(b);

    // keys each of this lane's rows sees; the fewest and the most of the wave's
    const int row_end = min(row0 + ROWS, n_rows);
    auto seen = [&](int row) { return p.causal ? max(0, len - n + 1 + row / p.G) : len; };
    int lim[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) lim[i] = seen(min(row0 + 16 * i + rr, n_rows - 1));
    const int lim_min = row0 < n_rows ? seen(row0) : 0, lim_max = row0 < n_rows ? seen(row_end - 1) : 0;

    // Q fragments
    bf16x8 qf[RT][HALF][2][NP];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int row = row0 + 16 * i + rr;
        const int t = row / p.G, h = kvh * p.G + row % p.G;
        const long at = (p.ts.tok_start ? (t_first + t) * p.q.sT : (long)b * p.q.sB + (long)t * p.q.sT) + (long)h * p.q.sH + g4 * 16;
#pragma unroll
        for (int hf = 0; hf < HALF; ++hf)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if constexpr (NP == 1) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (row < n_rows) w = *(const uint4*)((const T*)p.q.data + at + hf * 64 + s * 8);
                    const unsigned flip = p.neg | p.neg >> 16;
                    w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
                    qf[i][hf][s][0] = __builtin_bit_cast(bf16x8, w);
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = row < n_rows ? to_f32<T>(((const T*)p.q.data)[at + hf * 64 + s * 8 + e]) : 0.f;
                        x[e] = __uint_as_float(__float_as_uint(x[e]) ^ p.neg);
                    }
                    planes<NP>(x, qf[i][hf][s]);
                }
            }
    }

    f32x4 o[RT][D / 16];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[i][d] = f32x4{0, 0, 0, 0};
    }

    // blocks of 64 keys of this split, dealt to the waves
    const int blocks = (lim_max >> 6) + ((lim_max & 63) ? 1 : 0);
    const int per = (blocks + p.n_split - 1) / p.n_split;
    const int blk1 = min(blocks, (split + 1) * per);
    const long page_bytes = (long)c.P * D;
    const int k_group = 16 * (rr >> 2), k_in = rr & 3;     // 16-key group and place in it of this lane's K rows
    uint4 kf[4][HALF], vf[D / 16];
    float ks, vs;
    int pk, pv;                                            // pages of this lane's K rows and of its 16 keys of V (alike from 64 tokens a page)
    auto pages_of = [&](int blk) {
        pv = kv8_page(c, b, ((blk << 6) + 16 * g4) >> c.log2P);
        pk = c.P < 64 ? kv8_page(c, b, ((blk << 6) + k_group) >> c.log2P) : pv;
    };
    auto load_k = [&](int blk) {
        const uint8_t* kp = c.k + ((long)max(pk, 0) * c.Hkv + kvh) * page_bytes + ((((blk << 6) + k_group) & (c.P - 1)) + k_in) * D + g4 * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf) kf[t][hf] = ld_codes<(WR == 1)>(kp + t * 4 * D + hf * 64);
        ks = c.ks[(long)max(pv, 0) * c.Hkv + kvh];
    };
    auto load_v = [&](int blk) {
        const uint8_t* vp = c.v + ((long)max(pv, 0) * c.Hkv + kvh) * page_bytes + rr * c.P + (((blk << 6) + 16 * g4) & (c.P - 1));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) vf[d] = ld_codes<(WR == 1)>(vp + d * 16 * c.P);
        vs = c.vs[(long)max(pv, 0) * c.Hkv + kvh];
    };
    int blk = split * per + wk;
    if (blk < blk1) {
        pages_of(blk);
        load_k(blk);
        load_v(blk);
    }
    for (; blk < blk1; blk += WK) {
        const int j0 = blk << 6, jv = j0 + 16 * g4;
        const bool mask = lim_min - j0 < 64, more = blk + WK < blk1;
        const float nan = __uint_as_float(0x7fc00000u);
        const float kscale = pv < 0 ? nan : ks * p.scale2;
        if (more) pages_of(blk + WK);

        f32x4 st[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) st[i][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf) {
                const bf16x8 a0 = codes8<F>(kf[t][hf].x, kf[t][hf].y), a1 = codes8<F>(kf[t][hf].z, kf[t][hf].w);
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int pl = NP - 1; pl >= 0; --pl) {
                        st[i][t] = mfma(a0, qf[i][hf][0][pl], st[i][t]);
                        st[i][t] = mfma(a1, qf[i][hf][1][pl], st[i][t]);
                    }
            }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_k(blk + WK);          // in flight under the softmax and P.V
        __builtin_amdgcn_sched_barrier(0);

        // a block of zeros (scale 0) has codes of zero: any scale does.  The V scale rides in the exponent: p' = p * vs costs nothing per
        // element, the sum is divided by it once per block (the rounding of log2(vs) adds |log2 vs| 2^-24 to an element)
        const float vsc = vs == 0.f ? 1.f : vs, lv = __builtin_amdgcn_logf(vsc), iv = __builtin_amdgcn_rcpf(vsc);
        bf16x8 pf[RT][2][NP];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int left = lim[i] - jv;          // keys of this lane's 16 that the row sees
            if (mask) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * t + e >= left) st[i][t][e] = -INFINITY;
            }
            float mx = fmaxf(st[i][0][0], st[i][0][1]);
#pragma unroll
            for (int k = 2; k < 16; k += 2) mx = fmaxf(fmaxf(mx, st[i][k >> 2][k & 3]), st[i][k >> 2][(k & 3) + 1]);
            mx *= kscale;
            if (mask && left <= 0) mx = -INFINITY;      // nothing of these 16 keys is seen, and the scale may be any leftover
            mx = across_groups_max(mx);
            const float mn = fmaxf(m[i], mx);
            const float base = mn == -INFINITY ? 0.f : mn;
            if (__any(mn != m[i])) {
                const float alpha = __builtin_amdgcn_exp2f(m[i] - base);
                l[i] *= alpha;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[i][d] *= alpha;
                m[i] = mn;
            }
            const float nb = lv - base;
            float x[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = __builtin_amdgcn_exp2f(fmaf(st[i][k >> 2][k & 3], kscale, nb));
            if (mask) {                            // a scale behind the end may be NaN
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (k >= left) x[k] = 0.f;
            }
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) sum += x[k];
            // (a poisoned scale of a block that is seen shows in the sum)
            if (!mask || left > 0) l[i] = fmaf(sum, iv, l[i]);
            planes<NP>(x, pf[i][0]);
            planes<NP>(x + 8, pf[i][1]);
        }
        if (mask) {      // leftovers behind the sequence's end may hold NaN, which a probability of 0 does not silence
            const int keep = max(0, min(16, len - jv));
#pragma unroll
            for (int d = 0; d < D / 16; ++d) vf[d] = first_bytes(vf[d], keep);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const bf16x8 a0 = codes8<F>(vf[d].x, vf[d].y), a1 = codes8<F>(vf[d].z, vf[d].w);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int pl = NP - 1; pl >= 0; --pl) {
                    o[i][d] = mfma(a0, pf[i][0][pl], o[i][d]);
                    o[i][d] = mfma(a1, pf[i][1][pl], o[i][d]);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v(blk + WK);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        l[i] += __shfl_xor(l[i], 16, 64);
        l[i] += __shfl_xor(l[i], 32, 64);
    }

    // join the waves that shared the keys
    if constexpr (WK > 1) {
        const int R = p.lds_rows;
        float* sm = lds + (long)wr * WK * R * (D + 2);                    // [WK][R] m, [WK][R] l, [WK][R][D]
        float* sl = sm + WK * R;
        float* so = sl + WK * R;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = 16 * i + rr;
            if (r >= R) continue;
            if (g4 == 0) { sm[wk * R + r] = m[i]; sl[wk * R + r] = l[i]; }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                float* at = so + ((long)wk * R + r) * D + d * 16 + g4 * 4;
                at[0] = o[i][d][0]; at[1] = o[i][d][1]; at[2] = o[i][d][2]; at[3] = o[i][d][3];
            }
        }
        __syncthreads();
        for (int e = (wk * 64 + lane) * 4; e < (row_end - row0) * D; e += 64 * WK * 4) {
            const int r = e / D, d = e % D;
            float M = -INFINITY, L = 0.f;
            f32x4 acc = {0, 0, 0, 0};
            for (int w = 0; w < WK; ++w) M = fmaxf(M, sm[w * R + r]);
            for (int w = 0; w < WK; ++w) {
                // a wave without a finite score has a sum of 0, or NaN where it met a NaN
                const float mw = sm[w * R + r], f = mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - M);
                L += sl[w * R + r] * f;
                const float* x = so + ((long)w * R + r) * D + d;
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] += x[k] * f;
            }
            store_row<T, D>(p, b, t_first, kvh, row0 + r, d, split, M, L, acc);
        }
    } else {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = row0 + 16 * i + rr;
            if (row < n_rows)
#pragma unroll
                for (int d = 0; d < D / 16; ++d) store_row<T, D>(p, b, t_first, kvh, row, d * 16 + g4 * 4, split, m[i], l[i], o[i][d]);
        }
    }
}

// joins the splits: a wave per (token, head)
template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(AttnArgs p)
{
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6), row = w / p.H;
    const int h = (int)(w % p.H);
    if (row >= p.ts.N) return;
    long oat = row * p.o.sT;
    if (p.ts.tok_start) {
        if (row < p.ts.tok_start[0] || row >= p.ts.tok_start[p.ts.B]) return;
    } else {
        oat = row / p.ts.T * p.o.sB + row % p.ts.T * p.o.sT;
    }
    const float* part = p.part + w * p.n_split * (D + 4);
    float M = -INFINITY, L = 0.f, acc[D / 64] = {};
    for (int s = 0; s < p.n_split; ++s) M = fmaxf(M, part[s * (D + 4) + D]);
    for (int s = 0; s < p.n_split; ++s) {
        const float* x = part + s * (D + 4);
        const float ms = x[D], ls = x[D + 1];
        const float f = ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ms - M);
        L += ls * f;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) acc[k] += x[k * 64 + lane] * f;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int k = 0; k < D / 64; ++k) ((T*)p.o.data)[oat + (long)h * p.o.sH + k * 64 + lane] = from_f32<T>(acc[k] * inv);
    if (p.lse && lane == 0) p.lse[row * p.H + h] = L == 0.f ? -INFINITY : M * LN2 + logf(L);
}

// ---- host side --------------------------------------------------------------------------------------
#define RUN(x)                   \
    do {                         \
        const int rc__ = (x);    \
        if (rc__) return rc__;   \
    } while (0)

int log2_page(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : page == 256 ? 8 : -1; }

int check_cache(const char* fn, const uw_kv8_cache* c)
{
    UW_REQUIRE(c && c->k && c->v && c->k_scale && c->v_scale, "%s: null cache", fn);
    UW_REQUIRE(c->format == UW_KV8_INT8 || c->format == UW_KV8_E4M3, "%s: unknown code format %d", fn, c->format);
    UW_REQUIRE(log2_page(c->page) > 0, "%s: a page holds 16, 32, 64, 128 or 256 tokens, not %d", fn, c->page);
    UW_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim 64 or 128, not %d", fn, c->head_dim);
    UW_REQUIRE(c->n_pages > 0 && c->n_kv_heads > 0 && c->n_kv_heads <= 65535, "%s: %d pages of %d heads", fn, c->n_pages, c->n_kv_heads);
    UW_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0 && (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) == 0,
               "%s: cache arrays must be 16-byte aligned (scales 4)", fn);
    return UW_OK;
}

int check_seqs(const char* fn, const uw_kv8_seqs* t)
{
    UW_REQUIRE(t->dtype == UW_DTYPE_F32 || t->dtype == UW_DTYPE_BF16, "%s: dtype must be f32 or bf16", fn);
    UW_REQUIRE(t->B > 0 && t->n_tok >= 0, "%s: %d sequences, %lld rows", fn, t->B, (long long)t->n_tok);
    UW_REQUIRE(t->tok_start || (t->T >= 0 && t->n_tok == (int64_t)t->B * t->T), "%s: %lld rows are not %d x %d", fn,
               (long long)t->n_tok, t->B, t->T);
    UW_REQUIRE(t->n_tok <= 0x7fffffff, "%s: too many rows", fn);
    UW_REQUIRE(t->table && t->len && t->table_width > 0, "%s: null page table or lengths, or no columns", fn);
    UW_REQUIRE(t->table_width <= (1 << 23), "%s: %d table columns", fn, t->table_width);
    return UW_OK;
}

int check_tokens(const char* fn, const char* what, const uw_kv8_tokens* t, const uw_kv8_seqs* q)
{
    const int unit = q->dtype == UW_DTYPE_F32 ? 4 : 8;      // elements in 16 bytes
    UW_REQUIRE(q->n_tok == 0 || t->data, "%s: %s: null data", fn, what);
    UW_REQUIRE(((uintptr_t)t->data & 15) == 0 && t->seq_stride % unit == 0 && t->tok_stride % unit == 0 && t->head_stride % unit == 0,
               "%s: %s: base and strides must be multiples of 16 bytes", fn, what);
    return UW_OK;
}

Kv8View view_of(const uw_kv8_cache* c, const uw_kv8_seqs* q)
{
    Kv8View v;
    v.k = (uint8_t*)c->k;
    v.v = (uint8_t*)c->v;
    v.ks = c->k_scale;
    v.vs = c->v_scale;
    v.n_pages = c->n_pages;
    v.Hkv = c->n_kv_heads;
    v.P = c->page;
    v.log2P = log2_page(c->page);
    v.D = c->head_dim;
    v.table = q->table;
    v.width = q->table_width;
    return v;
}

TokArg arg_of(const uw_kv8_tokens* t) { return TokArg{t->data, (long)t->seq_stride, (long)t->tok_stride, (long)t->head_stride}; }
TokSpan span_of(const uw_kv8_seqs* t) { return TokSpan{t->tok_start, t->B, t->T, (long)t->n_tok}; }

// upper bound of the blocks a call touches, known without reading the lengths: n tokens touch at most (n - 1) / P + 2
long touched_bound(const uw_kv8_seqs* t, int P)
{
    if (t->tok_start) return t->n_tok / P + 2l * std::min((long)t->B, (long)t->n_tok);
    return (long)t->B * ((t->T + P - 2) / P + 1);
}

#define KV8_DISPATCH(format, dtype, CALL)                                                   \
    do {                                                                                    \
        if (format == UW_KV8_INT8) {                                                        \
            if (dtype == UW_DTYPE_BF16) { CALL(UW_KV8_INT8, bf16_t); } else { CALL(UW_KV8_INT8, float); } \
        } else {                                                                            \
            if (dtype == UW_DTYPE_BF16) { CALL(UW_KV8_E4M3, bf16_t); } else { CALL(UW_KV8_E4M3, float); } \
        }                                                                                   \
    } while (0)

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

int check_attention(const char* fn, const uw_kv8_attention_args* a)
{
    UW_REQUIRE(a, "%s: null arguments", fn);
    RUN(check_cache(fn, &a->cache));
    RUN(check_seqs(fn, &a->seqs));
    RUN(check_tokens(fn, "q", &a->q, &a->seqs));
    RUN(check_tokens(fn, "o", &a->o, &a->seqs));
    UW_REQUIRE(a->n_heads > 0 && a->n_heads % a->cache.n_kv_heads == 0, "%s: %d query heads over %d kv heads", fn, a->n_heads, a->cache.n_kv_heads);
    return UW_OK;
}

struct AttnPlan {
    int rt, wk, wr;      // row tiles of 16 per wave, waves sharing keys, waves side by side on rows
    int n_split, tiles, lds_rows;
    long groups, ws_bytes;
};

// How a call is cut.  Few rows per sequence: the waves of a workgroup share the keys, and the keys are cut over workgroups until
// the chip is full.  Many rows: the waves take rows of their own.
AttnPlan plan_attention(const uw_kv8_attention_args* a)
{
    AttnPlan p;
    const uw_kv8_cache* c = &a->cache;
    const int G = a->n_heads / c->n_kv_heads, B = a->seqs.B, T = a->seqs.tok_start ? 0 : a->seqs.T, width = a->seqs.table_width;
    const int64_t n_tok = a->seqs.n_tok;
    const long rows = T > 0 ? (long)T * G : (long)ceil_div(n_tok, B) * G;     // per sequence; packed: on average
    const int max_rt = 2;
    if (rows <= 16 * max_rt * 2) {
        p.rt = rows <= 16 ? 1 : 2;
        p.wk = 4;
        p.wr = 1;
    } else {
        p.rt = 2;
        p.wk = 1;
        p.wr = 4;
    }
    const int per = 16 * p.rt * p.wr;
    p.lds_rows = T > 0 ? (int)std::min((long)16 * p.rt, rows) : 16 * p.rt;
    p.tiles = T > 0 ? ceil_div(rows, per) : 0;
    p.groups = T > 0 ? (long)B * p.tiles : n_tok * G / per + std::min((long)B, (long)n_tok);
    const long blocks = ceil_div((long)width * c->page, 64);
    const long want = ceil_div(512, p.groups * c->n_kv_heads);
    p.n_split = (int)std::max(1l, std::min(std::min(want, 64l), (long)ceil_div(blocks, p.wk)));
    p.ws_bytes = p.n_split > 1 ? n_tok * a->n_heads * (int64_t)p.n_split * (c->head_dim + 4) * 4 : 0;
    return p;
}

template <int F, typename T, int D, int RT, int WK, int WR> int launch_attention_as(const AttnArgs& a, const AttnPlan& p, hipStream_t s)
{
    const size_t lds = WK > 1 ? (size_t)WR * WK * p.lds_rows * (D + 2) * 4 : 0;
    const dim3 grid((unsigned)(p.groups * a.c.Hkv * p.n_split));
    hipLaunchKernelGGL((kv8_attention_kernel<F, T, D, RT, WK, WR>), grid, dim3(64 * WK * WR), lds, s, a);
    UW_LAUNCH_CHECK();
    return UW_OK;
}

template <int F, typename T, int D> int launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t s)
{
    int rc;
    if (p.wr == 4) rc = launch_attention_as<F, T, D, 2, 1, 4>(a, p, s);
    else if (p.rt == 1) rc = launch_attention_as<F, T, D, 1, 4, 1>(a, p, s);
    else rc = launch_attention_as<F, T, D, 2, 4, 1>(a, p, s);
    if (rc || p.n_split == 1) return rc;
    hipLaunchKernelGGL((kv8_join_kernel<T, D>), dim3(ceil_div(a.ts.N * a.H, 4)), dim3(256), 0, s, a);
    UW_LAUNCH_CHECK();
    return UW_OK;
}

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

int64_t uw_kv8_attention_workspace_bytes(const uw_kv8_attention_args* a)
{
    if (check_attention("uw_kv8_attention_workspace_bytes", a)) return -1;
    return a->seqs.n_tok ? plan_attention(a).ws_bytes : 0;
}

int uw_kv8_attention(const uw_kv8_attention_args* a, void* stream)
{
    RUN(check_attention("uw_kv8_attention", a));
    const uw_kv8_seqs& q = a->seqs;
    if (q.n_tok == 0) return UW_OK;
    const AttnPlan pl = plan_attention(a);
    UW_REQUIRE(pl.ws_bytes == 0 || (a->ws && ((uintptr_t)a->ws & 15) == 0 && a->ws_bytes >= pl.ws_bytes),
               "uw_kv8_attention: workspace missing, misaligned or smaller than %lld bytes", (long long)pl.ws_bytes);
    UW_REQUIRE(pl.groups * a->cache.n_kv_heads * pl.n_split < (1 << 24) && q.n_tok * a->n_heads <= 0x7fffffff, "uw_kv8_attention: too many rows");
    AttnArgs x;
    x.c = view_of(&a->cache, &q);
    x.ts = span_of(&q);
    x.q = arg_of(&a->q);
    x.o = arg_of(&a->o);
    x.lse = a->lse;
    x.kv_len = q.len;
    x.part = (float*)a->ws;
    x.H = a->n_heads;
    x.G = a->n_heads / a->cache.n_kv_heads;
    x.causal = a->causal;
    x.n_split = pl.n_split;
    x.tiles = pl.tiles;
    x.groups = (int)pl.groups;
    x.lds_rows = pl.lds_rows;
    x.scale2 = fabsf(a->scale) * LOG2E;
    x.neg = a->scale < 0.f ? 0x80000000u : 0u;
#define CALL(F, T) RUN((a->cache.head_dim == 64 ? launch_attention<F, T, 64>(x, pl, (hipStream_t)stream) : launch_attention<F, T, 128>(x, pl, (hipStream_t)stream)))
    KV8_DISPATCH(a->cache.format, q.dtype, CALL);
#undef CALL
    return UW_OK;
}

}  // extern "C"
