// The 8-bit paged key/value cache: layout, code conversions and the bookkeeping shared by its kernels.
//
// A page ("block") holds P tokens (16 .. 256, a power of two) of every kv head.  Per head: K codes row by row [P][D], V codes
// transposed [D][P].  Both are then read along the index the attention product sums over -- D for q.k, the tokens for p.v -- as
// 16-byte chunks that are MFMA operands as they lie, with no transpose between memory and register.  One f32 scale per page, head
// and half; value = code * scale.  Two code formats, both exact in bf16 (8 significant bits):
//   int8  codes -127 .. 127, scale = largest |x| times the f32 next to 1/127
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
    int N;                      // rows altogether
    __device__ __forceinline__ long first(int b) const { return tok_start ? (long)tok_start[b] : (long)b * T; }
    // tokens of sequence b; a malformed tok_start gives 0 rather than rows outside [0, N)
    __device__ __forceinline__ int count(int b) const
    {
        if (!tok_start) return T;
        const int s = tok_start[b], e = tok_start[b + 1];
        return (s < 0 || e > N || e < s) ? 0 : e - s;
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

template <int F> __device__ __forceinline__ void kv8_decode4(unsigned w, float* x);
template <> __device__ __forceinline__ void kv8_decode4<UW_KV8_INT8>(unsigned w, float* x)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
}
template <> __device__ __forceinline__ void kv8_decode4<UW_KV8_E4M3>(unsigned w, float* x)
{
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
}

// byte j of word i <-> byte i of word j
__device__ __forceinline__ void transpose4(unsigned* w)
{
    const unsigned a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
    const unsigned c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302);
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
    if (F == UW_KV8_INT8) return fmaxf(amax * (1.0f / 127.0f), 0x1p-126f);      // a product, as tensor libraries divide by a constant on GPUs
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

struct TokArg {
    void* data;
    long sB, sT, sH;
};

// sums of lanes 0 .. own, in the vector ALU (row shifts, then the rows' totals handed on)
__device__ __forceinline__ int wave_scan(int x)
{
#define KV8_SCAN_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, true)
    KV8_SCAN_STEP(0x111, 0xf);
    KV8_SCAN_STEP(0x112, 0xf);
    KV8_SCAN_STEP(0x114, 0xf);
    KV8_SCAN_STEP(0x118, 0xf);
    KV8_SCAN_STEP(0x142, 0xa);
    KV8_SCAN_STEP(0x143, 0xc);
#undef KV8_SCAN_STEP
    return x;
}

// The idx-th (sequence, part) pair of a call, parts counted over the sequences in order; false past the last one.  cnt(b) = parts of
// sequence b.  Every wave works it out for itself: 256 sequences per step, four to a lane so that their lengths are asked for at
// once, and one scan.
template <typename CNT> __device__ __forceinline__ bool locate(int idx, int B, CNT cnt, int& b_out, int& j_out)
{
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += 256) {
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = 0;
        const int first = b0 + lane * 4;
        if (first < B) {
#pragma unroll
            for (int i = 0; i < 4; ++i) n[i] = cnt(min(first + i, B - 1));
#pragma unroll
            for (int i = 1; i < 4; ++i) n[i] = first + i < B ? n[i] : 0;
        }
        const int own = (n[0] + n[1]) + (n[2] + n[3]), incl = wave_scan(own);
        const unsigned long long over = __ballot(base + incl > idx);
        if (over) {
            const int w = __ffsll((long long)over) - 1;
            int j = idx - base - __builtin_amdgcn_readlane(incl - own, w), b = b0 + w * 4;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const int c = __builtin_amdgcn_readlane(n[i], w);
                if (b == b0 + w * 4 + i && j >= c) { j -= c; ++b; }
            }
            b_out = b;
            j_out = j;
            return true;
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// The idx-th (sequence, part) pair when parts are dealt round by round from the sequences' ends: every sequence's last part, then every
// second to last one, ...  (of causal queries the last parts are the longest).  Up to 256 sequences; j_out counts from the end.
template <typename CNT> __device__ __forceinline__ bool locate_from_end(int idx, int B, CNT cnt, int& b_out, int& j_out)
{
    const int lane = threadIdx.x & 63;
    int n[4] = {0, 0, 0, 0}, most = 0;
    if (lane * 4 < B) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = cnt(min(lane * 4 + i, B - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (lane * 4 + i >= B) n[i] = 0;
            most = max(most, n[i]);
        }
    }
    most = (int)across_wave((unsigned)most, [](unsigned p, unsigned q) { return max(p, q); });
    // parts of the first r rounds
    auto dealt = [&](int r) { return __builtin_amdgcn_readlane(wave_scan((min(n[0], r) + min(n[1], r)) + (min(n[2], r) + min(n[3], r))), 63); };
    if (dealt(most) <= idx) return false;
    int lo = 0, hi = most;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (dealt(mid) <= idx) lo = mid;
        else hi = mid;
    }
    int k = idx - dealt(lo);
    const int own = (n[0] > lo) + (n[1] > lo) + (n[2] > lo) + (n[3] > lo), incl = wave_scan(own);
    const int w = __ffsll((long long)__ballot(incl > k)) - 1;
    k -= __builtin_amdgcn_readlane(incl - own, w);
    int b = w * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int has = __builtin_amdgcn_readlane(n[i], w) > lo ? 1 : 0;
        if (has && k == 0) b_out = b + i;
        k -= has;
    }
    b_out = __builtin_amdgcn_readfirstlane(b_out);
    j_out = lo;
    return true;
}

// ---- host side: what every entry checks -----------------------------------------------------------------
#define RUN(x)                   \
    do {                         \
        const int rc__ = (x);    \
        if (rc__) return rc__;   \
    } while (0)

static inline int log2_page(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : page == 256 ? 8 : -1; }

static inline int check_cache(const char* fn, const uw_kv8_cache* c)
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

static inline int check_seqs(const char* fn, const uw_kv8_seqs* t)
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

static inline int check_tokens(const char* fn, const char* what, const uw_kv8_tokens* t, const uw_kv8_seqs* q)
{
    const int unit = q->dtype == UW_DTYPE_F32 ? 4 : 8;      // elements in 16 bytes
    UW_REQUIRE(q->n_tok == 0 || t->data, "%s: %s: null data", fn, what);
    UW_REQUIRE(((uintptr_t)t->data & 15) == 0 && t->seq_stride % unit == 0 && t->tok_stride % unit == 0 && t->head_stride % unit == 0,
               "%s: %s: base and strides must be multiples of 16 bytes", fn, what);
    return UW_OK;
}

static inline Kv8View view_of(const uw_kv8_cache* c, const uw_kv8_seqs* q)
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

static inline TokArg arg_of(const uw_kv8_tokens* t) { return TokArg{t->data, (long)t->seq_stride, (long)t->tok_stride, (long)t->head_stride}; }
static inline TokSpan span_of(const uw_kv8_seqs* t) { return TokSpan{t->tok_start, t->B, t->T, (int)t->n_tok}; }

#define KV8_DISPATCH(format, dtype, CALL)                                                   \
    do {                                                                                    \
        if (format == UW_KV8_INT8) {                                                        \
            if (dtype == UW_DTYPE_BF16) { CALL(UW_KV8_INT8, bf16_t); } else { CALL(UW_KV8_INT8, float); } \
        } else {                                                                            \
            if (dtype == UW_DTYPE_BF16) { CALL(UW_KV8_E4M3, bf16_t); } else { CALL(UW_KV8_E4M3, float); } \
        }                                                                                   \
    } while (0)
