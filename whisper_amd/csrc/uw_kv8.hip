// The 8-bit paged key/value cache: append, read back, attention.
#include "../../include/uw_hip.h"
#include "uw_kv8.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

// One element of a token array, widened.
template <typename T> __device__ __forceinline__ float ld_elem(const void* p, long at) { return to_f32<T>(((const T*)p)[at]); }

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

template <int F, typename T>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8View c, TokSpan ts, TokArg ka, TokArg va, const int32_t* pos_of)
{
    __shared__ unsigned s_max[4];
    int b, j;
    if (!locate(blockIdx.x, ts.B, [&](int i) { return touched(pos_of[i], ts.count(i), c.log2P); }, b, j)) return;
    const bool is_v = blockIdx.z;
    const int h = blockIdx.y, tid = threadIdx.x, P = c.P, D = c.D;
    const int pos = pos_of[b], n = ts.count(b);
    const long blk = (pos >> c.log2P) + j, p0 = blk << c.log2P;      // first position of the block
    const int page = kv8_page(c, b, blk);
    if (page < 0) return;
    const int t0 = (int)max(0l, p0 - pos), t1 = (int)min((long)n, p0 + P - pos);   // tokens of the call in this block
    const int r0 = (int)(pos + t0 - p0);                                            // their first row in the block = earlier tokens
    const TokArg& a = is_v ? va : ka;
    const long src = (ts.tok_start ? ts.first(b) * a.sT : (long)b * a.sB) + h * a.sH + (long)t0 * a.sT;
    uint8_t* codes = (is_v ? c.v : c.k) + ((long)page * c.Hkv + h) * P * D;
    float* scale = (is_v ? c.vs : c.ks) + (long)page * c.Hkv + h;
    const int rows = t1 - t0, ne = rows * D;

    // largest |x| by its bits: they order like the values, with infinity and NaN above every number
    unsigned mx = 0;
    for (int e = tid; e < ne; e += 256)
        mx = max(mx, __float_as_uint(ld_elem<T>(a.data, src + (long)(e / D) * a.sT + e % D)) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
    if ((tid & 63) == 0) s_max[tid >> 6] = mx;
    const float old_s = *scale;
    __syncthreads();
    mx = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    const float amax = __uint_as_float(mx);
    float s;
    int grow = 0;
    if (mx >= 0x7f800000u || (r0 > 0 && !(fabsf(old_s) < INFINITY))) {
        s = __uint_as_float(0x7fc00000u);
    } else if (r0 == 0 || old_s <= 0.f) {
        s = kv8_base_scale<F>(amax);
    } else {
        grow = kv8_growth<F>(amax, old_s);
        s = ldexpf(old_s, grow);
    }
    if (grow) {
        const float down = ldexpf(1.f, -grow);
        for (int e = tid; e < r0 * D; e += 256) {
            const int r = e / D, d = e % D;
            uint8_t* at = codes + (is_v ? d * P + r : r * D + d);
            *at = kv8_encode<F>(kv8_decode<F>(*at), down);
        }
    }
    const float rs = s > 0.f ? 1.0f / s : 0.f;
    for (int e = tid; e < ne; e += 256) {
        const int r = e / D, d = e % D;
        const uint8_t code = rs > 0.f ? kv8_encode<F>(ld_elem<T>(a.data, src + (long)r * a.sT + d), rs) : 0;
        codes[is_v ? d * P + r0 + r : (r0 + r) * D + d] = code;
    }
    if (tid == 0) *scale = s;
}

template <int F, typename T>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8View c, TokSpan ts, TokArg ka, TokArg va, const int32_t* first_of)
{
    int b, j;
    if (!locate(blockIdx.x, ts.B, [&](int i) { return touched(first_of[i], ts.count(i), c.log2P); }, b, j)) return;
    const bool is_v = blockIdx.z;
    const int h = blockIdx.y, tid = threadIdx.x, P = c.P, D = c.D;
    const int pos = first_of[b], n = ts.count(b);
    const long blk = (pos >> c.log2P) + j, p0 = blk << c.log2P;
    const int page = kv8_page(c, b, blk);
    const int t0 = (int)max(0l, p0 - pos), t1 = (int)min((long)n, p0 + P - pos);
    const int r0 = (int)(pos + t0 - p0);
    const TokArg& a = is_v ? va : ka;
    const long dst = (ts.tok_start ? ts.first(b) * a.sT : (long)b * a.sB) + h * a.sH + (long)t0 * a.sT;
    const uint8_t* codes = (is_v ? c.v : c.k) + ((long)max(page, 0) * c.Hkv + h) * P * D;
    const float s = page < 0 ? __uint_as_float(0x7fc00000u) : (is_v ? c.vs : c.ks)[(long)page * c.Hkv + h];
    for (int e = tid; e < (t1 - t0) * D; e += 256) {
        const int r = e / D, d = e % D;
        const float v = page < 0 ? 0.f : kv8_decode<F>(codes[is_v ? d * P + r0 + r : (r0 + r) * D + d]);
        ((T*)a.data)[dst + (long)r * a.sT + d] = from_f32<T>(v * s);
    }
}

// attention, one workgroup per query row and head: 256 keys per round, a lane scores one key; then a lane owns one output element
template <int F, typename T>
__global__ __launch_bounds__(256) void kv8_attention_kernel(Kv8View c, TokSpan ts, TokArg qa, TokArg oa, float* lse, int H,
                                                            const int32_t* kv_len, int causal, float scale)
{
    __shared__ float q[128], p_s[256], red[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.y, D = c.D;
    const long row = blockIdx.x;
    int b = 0, t = 0;
    if (ts.tok_start) {
        for (int i = 0; i < ts.B; ++i)
            if (ts.count(i) > 0 && row >= ts.tok_start[i] && row < ts.tok_start[i + 1]) { b = i; t = (int)(row - ts.tok_start[i]) + 1; }
        if (!t) return;
        --t;
    } else {
        b = (int)(row / ts.T);
        t = (int)(row % ts.T);
    }
    const int g = h / (H / c.Hkv);
    const long base = ts.tok_start ? row * qa.sT : (long)b * qa.sB + (long)t * qa.sT;
    const long obase = ts.tok_start ? row * oa.sT : (long)b * oa.sB + (long)t * oa.sT;
    const long n_keys = causal ? max(0l, (long)kv_len[b] - ts.count(b) + t + 1) : max(0, kv_len[b]);
    if (tid < D) q[tid] = ld_elem<T>(qa.data, base + h * qa.sH + tid) * scale;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (long k0 = 0; k0 < n_keys; k0 += 256) {
        __syncthreads();
        const long j = k0 + tid;
        float s = -INFINITY;
        if (j < n_keys) {
            const int page = kv8_page(c, b, j >> c.log2P);
            const long at = (long)max(page, 0) * c.Hkv + g;
            const uint8_t* kr = c.k + (at * c.P + (j & (c.P - 1))) * D;
            s = 0.f;
            for (int d = 0; d < D; ++d) s = fmaf(q[d], kv8_decode<F>(kr[d]), s);
            s = page < 0 ? __uint_as_float(0x7fc00000u) : s * c.ks[at];
        }
        const bool bad = __syncthreads_or(s != s);
        float mx = wave_max(s);
        if (lane == 0) red[wave] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        float mn = fmaxf(m, mx);
        if (bad) mn = __uint_as_float(0x7fc00000u);
        const float p = (j < n_keys) ? expf(s - mn) : 0.f;
        const float sum = wave_sum(p);
        __syncthreads();
        if (lane == 0) red[wave] = sum;
        p_s[tid] = p;
        __syncthreads();
        const float f = m == -INFINITY ? 0.f : expf(m - mn);
        l = l * f + ((red[0] + red[1]) + (red[2] + red[3]));
        acc *= f;
        m = mn;
        if (tid < D) {
            const int lim = (int)min(256l, n_keys - k0);
            for (int i = 0; i < lim; ++i) {
                const long jj = k0 + i;
                const int page = kv8_page(c, b, jj >> c.log2P);
                const long at = (long)max(page, 0) * c.Hkv + g;
                acc = fmaf(p_s[i] * c.vs[at], kv8_decode<F>(c.v[(at * D + tid) * c.P + (jj & (c.P - 1))]), acc);
            }
        }
    }
    if (tid < D) ((T*)oa.data)[obase + h * oa.sH + tid] = from_f32<T>(n_keys > 0 ? acc / l : 0.f);
    if (lse && tid == 0) lse[row * H + h] = n_keys > 0 ? m + logf(l) : -INFINITY;
}

// ---- host side --------------------------------------------------------------------------------------
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

int check_tokens(const char* fn, const char* what, const uw_kv8_tokens* t, int dtype)
{
    UW_REQUIRE(dtype == UW_DTYPE_F32 || dtype == UW_DTYPE_BF16, "%s: dtype must be f32 or bf16", fn);
    const int unit = dtype == UW_DTYPE_F32 ? 4 : 8;      // elements in 16 bytes
    UW_REQUIRE(t && t->B > 0 && t->n_tok >= 0, "%s: %s: %d sequences", fn, what, t ? t->B : 0);
    UW_REQUIRE(t->n_tok == 0 || t->data, "%s: %s: null data", fn, what);
    UW_REQUIRE(t->tok_start || (t->T >= 0 && t->n_tok == (int64_t)t->B * t->T), "%s: %s: %lld rows are not %d x %d", fn, what,
               (long long)t->n_tok, t->B, t->T);
    UW_REQUIRE(t->n_tok <= 0x7fffffff, "%s: %s: too many rows", fn, what);
    UW_REQUIRE(((uintptr_t)t->data & 15) == 0 && t->seq_stride % unit == 0 && t->tok_stride % unit == 0 && t->head_stride % unit == 0,
               "%s: %s: base and strides must be multiples of 16 bytes", fn, what);
    return UW_OK;
}

int check_table(const char* fn, const int32_t* table, int width, const int32_t* len)
{
    UW_REQUIRE(table && len && width > 0, "%s: null page table or lengths, or no columns", fn);
    UW_REQUIRE(width <= (1 << 23), "%s: %d table columns", fn, width);
    return UW_OK;
}

int check_pair(const char* fn, const uw_kv8_tokens* k, const uw_kv8_tokens* v)
{
    UW_REQUIRE(k->tok_start == v->tok_start && k->B == v->B && k->n_tok == v->n_tok && (k->tok_start || k->T == v->T),
               "%s: k and v must hold the same tokens", fn);
    return UW_OK;
}

Kv8View view_of(const uw_kv8_cache* c, const int32_t* table, int width)
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
    v.table = table;
    v.width = width;
    return v;
}

TokArg arg_of(const uw_kv8_tokens* t) { return TokArg{t->data, (long)t->seq_stride, (long)t->tok_stride, (long)t->head_stride}; }
TokSpan span_of(const uw_kv8_tokens* t) { return TokSpan{t->tok_start, t->B, t->T, (long)t->n_tok}; }

// upper bound of the blocks a call touches, known without reading the lengths: n tokens touch at most (n - 1) / P + 2
long touched_bound(const uw_kv8_tokens* t, int P)
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

}  // namespace

#define RUN(x)                   \
    do {                         \
        const int rc__ = (x);    \
        if (rc__) return rc__;   \
    } while (0)

extern "C" {

int uw_kv8_append(const uw_kv8_cache* cache, int dtype, const uw_kv8_tokens* k, const uw_kv8_tokens* v, const int32_t* table,
                  int table_width, const int32_t* pos, void* stream)
{
    RUN(check_cache("uw_kv8_append", cache));
    RUN(check_tokens("uw_kv8_append", "k", k, dtype));
    RUN(check_tokens("uw_kv8_append", "v", v, dtype));
    RUN(check_pair("uw_kv8_append", k, v));
    RUN(check_table("uw_kv8_append", table, table_width, pos));
    if (k->n_tok == 0) return UW_OK;
    const Kv8View c = view_of(cache, table, table_width);
    const dim3 grid((unsigned)touched_bound(k, c.P), c.Hkv, 2);
#define CALL(F, T) hipLaunchKernelGGL((kv8_append_kernel<F, T>), grid, dim3(256), 0, (hipStream_t)stream, c, span_of(k), arg_of(k), arg_of(v), pos)
    KV8_DISPATCH(cache->format, dtype, CALL);
#undef CALL
    UW_LAUNCH_CHECK();
    return UW_OK;
}

int uw_kv8_read(const uw_kv8_cache* cache, int dtype, const uw_kv8_tokens* k, const uw_kv8_tokens* v, const int32_t* table,
                int table_width, const int32_t* first, void* stream)
{
    RUN(check_cache("uw_kv8_read", cache));
    RUN(check_tokens("uw_kv8_read", "k", k, dtype));
    RUN(check_tokens("uw_kv8_read", "v", v, dtype));
    RUN(check_pair("uw_kv8_read", k, v));
    RUN(check_table("uw_kv8_read", table, table_width, first));
    if (k->n_tok == 0) return UW_OK;
    const Kv8View c = view_of(cache, table, table_width);
    const dim3 grid((unsigned)touched_bound(k, c.P), c.Hkv, 2);
#define CALL(F, T) hipLaunchKernelGGL((kv8_read_kernel<F, T>), grid, dim3(256), 0, (hipStream_t)stream, c, span_of(k), arg_of(k), arg_of(v), first)
    KV8_DISPATCH(cache->format, dtype, CALL);
#undef CALL
    UW_LAUNCH_CHECK();
    return UW_OK;
}

int64_t uw_kv8_attention_workspace_bytes(const uw_kv8_cache* cache, int n_heads, int B, int64_t n_tok, int T, int table_width)
{
    return 0;
}

int uw_kv8_attention(const uw_kv8_cache* cache, int dtype, const uw_kv8_tokens* q, const uw_kv8_tokens* o, float* lse, int n_heads,
                     const int32_t* table, int table_width, const int32_t* kv_len, int causal, float scale, void* ws, void* stream)
{
    RUN(check_cache("uw_kv8_attention", cache));
    RUN(check_tokens("uw_kv8_attention", "q", q, dtype));
    RUN(check_tokens("uw_kv8_attention", "o", o, dtype));
    RUN(check_pair("uw_kv8_attention", q, o));
    RUN(check_table("uw_kv8_attention", table, table_width, kv_len));
    UW_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0, "uw_kv8_attention: %d query heads over %d kv heads", n_heads, cache->n_kv_heads);
    if (q->n_tok == 0) return UW_OK;
    const Kv8View c = view_of(cache, table, table_width);
    const dim3 grid((unsigned)q->n_tok, n_heads);
#define CALL(F, T) hipLaunchKernelGGL((kv8_attention_kernel<F, T>), grid, dim3(256), 0, (hipStream_t)stream, c, span_of(q), arg_of(q), arg_of(o), lse, n_heads, kv_len, causal, scale)
    KV8_DISPATCH(cache->format, dtype, CALL);
#undef CALL
    UW_LAUNCH_CHECK();
    return UW_OK;
}

}  // extern "C"
