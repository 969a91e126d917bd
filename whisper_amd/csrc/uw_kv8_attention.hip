// Attention over the 8-bit paged key/value cache.
#include "../../include/uw_hip.h"
#include "uw_kv8.h"
#include "uw_kernels.h"
#include <algorithm>
#include <type_traits>

namespace {

// ------------------------------------------------------------------------------------------------
// Attention.  Rows of one kv head are its G query heads of every query token, token-major: row = t * G + g.  A wave works on 64
// keys at a time and 16 * RT rows, in registers throughout:
//   S^T = K Q^T    16x16x32 MFMA, A = K codes as bf16 (exact), B = Q; lane (row = lane & 15, g = lane >> 4) gets for tile t the keys
//                  16 g + 4 t + 0..3, because row slot r of tile t holds key 16 (r >> 2) + 4 t + (r & 3)
//   O^T = V^T P^T  A = V codes as they lie (16 consecutive keys 16 g .. of one channel), B = P straight from those lanes
// so neither K nor V nor P passes through LDS.  K scales multiply the scores, V scales ride in the exponent of the weights; one per 16
// keys at least, so one per lane.  References, sums and outputs are f32.
//
// bf16 queries enter exactly, their weights as two bf16 planes: off by 2^-16 of each at most, with the whole of f32's exponent, so that
// a row has its result to the same error when its largest weights meet values of zero.  (One f16 plane, which is faster -- 145 us for the
// prompts below when this took 185, 2 to 4 % where the stream of codes bounds, 0.6 of 9.7 us for one window -- loses the weights below 2^-25
// of the largest and keeps them in the sum.)  f32 queries and weights enter as three planes (24 bits): the codes being exact in bf16, that
// is f32 arithmetic at a third of the bf16 rate.
//
// What bounds it: few rows of a head -- the stream of codes; 128 windows' token over 1500 keys of 12 heads, e4m3 (296 MB) 49.6 us, 6.0 TB/s;
// five tokens of 4 heads a kv head over long ragged tables (297 MB) 58 us, 5.1 TB/s, and 4.8 us for the join.  Many rows -- the vector ALU,
// which has a multiply-add, an exponential (a quarter of the rate), an addition and the two planes to do for each weight; it is at work in 72 %
// of the cycles, the matrix unit, with 192 or 384 multiply-adds for a weight, in 39 %, and LDS in 40 %, without bank conflicts: 33380 causal
// rows of 4 heads over 5000 keys 185 us, 585 TFLOP/s counted as 4 D operations a weight.  One window of 6 heads -- a chain of lengths, pages,
// codes, three blocks a wave and the join of eight waves: 9.7 us (e4m3 9.2).  170 f32 rows of 64 heads over 1500 keys: 24.4 us, 171
// TFLOP/s, three times that on the matrix unit.
//
// What a decoder step adds: one query token per window, its output in the operand layout of the product that follows, and the
// probabilities of the alignment heads.
struct StepArgs {
    const int32_t* active;       // [B]; 0: the window is finished, nothing is written (or null)
    void* out_lo;                // bf16: the plane of what rounding the output dropped (or null)
    int d;                       // heads * 64
    float* rows;                 // probabilities [B][slots][n_rows][S] (or null)
    long rows_sB, rows_sSel;
    const int32_t* row_index;    // [B] row to write, outside 0 .. n_rows-1: none
    int n_rows, S;
    signed char slot[32];        // per head, -1: not an alignment head
};

struct AttnArgs {
    Kv8View c;
    TokSpan ts;
    TokArg q, o;
    float* lse;
    const int32_t* kv_len;
    float* part;         // [rows][H][n_split][D + 4] partial results (output, its reference, sum, its reference) when n_split > 1
    int H, G, log2G, causal;   // log2G: -1 where G is no power of two
    int n_split;         // 1: an item is a row tile of a sequence; else at most so many items share a tile, each with a part of the keys
    int target, min_chunk;   // n_split > 1: items a head should come to, and the fewest blocks of 64 keys of one
    int tiles;           // row tiles per sequence (uniform)
    int max_blocks;      // blocks that the table can hold, and one more: a longer sequence sees a page that does not exist
    int lds_rows;        // rows of a tile that can be in use
    float scale2;        // |scale| * log2(e)
    unsigned neg;        // sign bit of scale, moved to the queries
    StepArgs step;
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

// The planes of 8 f32 values, each the rounded rest of those before.  DOT: the rest is taken from a packed pair by one dot product with
// (-1, 0) or (0, -1), exact like the subtraction that needs the part unpacked first.
template <int NP, bool DOT> __device__ __forceinline__ void planes(const float* x, bf16x8* out)
{
    unsigned own0 = 0x0000bf80u, own1 = 0xbf800000u;        // bf16 pairs (-1, 0), (0, -1)
    asm("" : "+s"(own0), "+s"(own1));                       // in registers: as an inline constant the first is read as the second
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a = x[e], b = x[e + 1];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const bf16x2 part = {(__bf16)a, (__bf16)b};
            out[n][e] = part[0];
            out[n][e + 1] = part[1];
            if (n + 1 == NP) continue;
            a = DOT ? __builtin_amdgcn_fdot2_f32_bf16(part, __builtin_bit_cast(bf16x2, own0), a, false) : a - (float)part[0];
            b = DOT ? __builtin_amdgcn_fdot2_f32_bf16(part, __builtin_bit_cast(bf16x2, own1), b, false) : b - (float)part[1];
        }
    }
}

// keeps the first n of 16 bytes
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n)
{
    auto m = [&](int k) { return k <= 0 ? 0u : k >= 4 ? ~0u : (1u << (8 * k)) - 1u; };
    return make_uint4(v.x & m(n), v.y & m(n - 4), v.z & m(n - 8), v.w & m(n - 12));
}

// ---- which workgroup does what ------------------------------------------------------------------------------------------
__device__ __forceinline__ int blocks_of(const AttnArgs& p, int b)
{
    const int len = max(0, p.kv_len[b]);
    return min((len >> 6) + ((len & 63) ? 1 : 0), p.max_blocks);
}
__device__ __forceinline__ int tiles_of(const AttnArgs& p, int b, int rows) { return p.ts.tok_start ? (int)(((long)p.ts.count(b) * p.G + rows - 1) / rows) : p.tiles; }

// Keys are cut by what is there, not by what the table could hold: the blocks of all sequences together, over the items wanted.  So
// unequal lengths give equal items, and a call over one long sequence as many as one over many short ones.
__device__ __forceinline__ int chunk_of(const AttnArgs& p, int rows)
{
    long sum = 0;
    for (int b = threadIdx.x & 63; b < p.ts.B; b += 64) sum += (long)tiles_of(p, b, rows) * blocks_of(p, b);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    return (int)max((long)p.min_chunk, (sum + p.target - 1) / p.target);
}
__device__ __forceinline__ int splits_of(const AttnArgs& p, int b, int chunk) { return max(1, (blocks_of(p, b) + chunk - 1) / chunk); }

// a 16-byte piece of the cache; ONCE: it need not stay in L2.  The shapes whose waves share the keys ask so: with one row tile of a head no
// other workgroup wants the piece.  With several they do, and ask again; what the hint does there has not been measured apart.
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

// op over WK (4 or 8) neighbouring lanes' values, where those of a row of sixteen repeat after WK lanes
template <int WK, typename OP> __device__ __forceinline__ float across_waves(float x, OP op)
{
#define KV8_ROTATED(n) x = op(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + n, 0xf, 0xf, true)))
    if constexpr (WK == 8) KV8_ROTATED(4);
    KV8_ROTATED(2);
    KV8_ROTATED(1);
#undef KV8_ROTATED
    return x;
}

// what a wave, a workgroup or an item knows of a row beside its output
struct RowState { float m, l, ms; };

// out = o * f0 * f1, f0 f1 = 2^(m - ms) / l in two steps: one alone runs out of exponent where all values are very small.  A row that saw
// no key has l = 0
__device__ __forceinline__ void result_of(const RowState& a, float& f0, float& f1, float& lse)
{
    f1 = __builtin_amdgcn_exp2f(0.5f * (a.m - a.ms));
    f0 = a.l == 0.f ? 0.f : f1 / a.l;
    if (a.l == 0.f) f1 = 0.f;
    lse = a.l == 0.f ? -INFINITY : a.ms * LN2 + logf(a.l);
}

// four channels of a finished row (or of a split's part of it)
template <typename T, int D>
__device__ __forceinline__ void store_row(const AttnArgs& p, int b, long t_first, int kvh, int row, int d, int split, int splits, RowState a, f32x4 acc)
{
    const int t = p.log2G >= 0 ? row >> p.log2G : row / p.G, h = kvh * p.G + row - t * p.G;
    const long rg = t_first + t;                        // row of the call
    if (splits > 1) {
        float* at = p.part + ((rg * p.H + h) * p.n_split + split) * (D + 4);
        *(f32x4*)(at + d) = acc;
        if (d == 0) { at[D] = a.m; at[D + 1] = a.l; at[D + 2] = a.ms; }
        return;
    }
    float f0, f1, lse;
    result_of(a, f0, f1, lse);
    T* out = (T*)p.o.data + (p.ts.tok_start ? rg * p.o.sT : (long)b * p.o.sB + (long)t * p.o.sT) + (long)h * p.o.sH + d;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = from_f32<T>(acc[k] * f0 * f1);
    *(T4*)out = v;
    if (p.lse && d == 0) p.lse[rg * p.H + h] = lse;
}

// WK waves share the keys of a row tile (their results are joined in LDS), WR row tiles per workgroup
//
// WR = 4: the four waves go through the same blocks together.  Each brings a quarter of a block's codes, turns them into operands and
// lays them in LDS in the order the lanes hold them, so that a code is converted once for 64 * RT rows; operands are read back as
// whole 1 KiB pieces, without bank conflicts.  Two buffers and one barrier a block: while block x is worked on, x + 1 is converted
// and the codes of x + 2 are under way in eight registers.
template <int F, typename T, int D, int RT, int WK, int WR, bool STEP>
__global__ __launch_bounds__(64 * WK * WR, (sizeof(T) == 2 && D == 64) ? (RT == 1 ? 4 : 3) : 2) void kv8_attention_kernel(AttnArgs p)
{
    constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NW = sizeof(T) == 4 ? 3 : 2;       // planes of a query and of a weight
    constexpr int ROWS = 16 * RT, HALF = D / 64;
    constexpr bool DOT = WR == 4 || NQ == 3;
    constexpr bool SHARE = WR == 4;
    constexpr int BUFFER = 64 * D * 4 / 16;            // SHARE: 16-byte pieces of a block's operands
    static_assert(WR == 1 || WK == 1, "waves share keys or stand side by side on rows");
    static_assert(WR == 1 || WR == 4, "");
    static_assert(!STEP || (D == 64 && RT == 1 && WK > 1), "a decoder step has one row of a head");
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wave % WK, wr = wave / WK;
    const int rr = lane & 15, g4 = lane >> 4;
    const Kv8View& c = p.c;

    // which kv head, sequence, rows and part of the keys.  Heads run fastest: a head's workgroups land on one XCD when their number
    // is a multiple of 8, and share its L2.  The last rows of all sequences come first: causal ones see most, and a long item that
    // starts late is waited for (4500, 2782 and 1063 tokens of 16 heads, with one f16 plane of weights: 187 us in the sequences' order, 156 so).
    int b, tile, split = 0, splits = 1, chunk = 0;
    const int kvh = blockIdx.x % c.Hkv, item = blockIdx.x / c.Hkv;
    if (p.n_split > 1) {
        int j;
        chunk = chunk_of(p, ROWS * WR);
        if (!locate(item, p.ts.B, [&](int i) { return tiles_of(p, i, ROWS * WR) * splits_of(p, i, chunk); }, b, j)) return;
        splits = splits_of(p, b, chunk);
        tile = j / splits;
        split = j % splits;
    } else if (p.ts.tok_start) {
        const auto count = [&](int i) { return tiles_of(p, i, ROWS * WR); };
        if (WR > 1 && p.ts.B <= 256) {
            if (!locate_from_end(item, p.ts.B, count, b, tile)) return;
            tile = count(b) - 1 - tile;
        } else {
            if (!locate(item, p.ts.B, count, b, tile)) return;
        }
    } else {
        b = item % p.ts.B;
        tile = p.tiles - 1 - item / p.ts.B;
    }
    // (the same in all lanes; in scalar registers what is kept over the loop spills nothing.  Not the first row of the side-by-side shape, nor the
    // chunk: the loop is then compiled with a hundred registers spilled)
    split = __builtin_amdgcn_readfirstlane(split);
    splits = __builtin_amdgcn_readfirstlane(splits);
    if (STEP && p.step.active && !p.step.active[b]) return;
    // STEP: an alignment head's scores are kept in LDS (behind what the waves join there) until their sum is known
    float *scores = nullptr, *row_out = nullptr;
    if constexpr (STEP) {
        const int slot = p.step.slot[kvh];
        if (p.step.rows && slot >= 0) {
            const int ri = p.step.row_index[b];
            if (ri >= 0 && ri < p.step.n_rows) {
                row_out = p.step.rows + (long)b * p.step.rows_sB + (long)slot * p.step.rows_sSel + (long)ri * p.step.S;
                scores = lds + WK * (D + 3);
            }
        }
    }
    const int n = p.ts.count(b), n_rows = n * p.G;
    const int row0 = SHARE ? (tile * WR + wr) * ROWS : __builtin_amdgcn_readfirstlane((tile * WR + wr) * ROWS);
    const int len = max(0, p.kv_len[b]);
    const long t_first = p.ts.first(b);

    // keys each of this lane's rows sees; the fewest and the most of the wave's
    const int row_end = min(row0 + ROWS, n_rows);
    auto token_of = [&](int row) { return p.log2G >= 0 ? row >> p.log2G : row / p.G; };
    auto seen = [&](int row) { return p.causal ? max(0, len - n + 1 + token_of(row)) : len; };
    int lim[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) lim[i] = seen(min(row0 + 16 * i + rr, n_rows - 1));
    const int lim_min = row0 < n_rows ? seen(row0) : 0, lim_max = row0 < n_rows ? seen(row_end - 1) : 0;

    // the queries' bytes are asked for here and made into fragments once the first codes are on their way too
    bf16x8 qf[RT][HALF][2][NQ];
    uint4 q_raw[RT][HALF][2][sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int row = row0 + 16 * i + rr, t = token_of(row), h = kvh * p.G + row - t * p.G;
        const T* from = (const T*)p.q.data + (p.ts.tok_start ? (t_first + t) * p.q.sT : (long)b * p.q.sB + (long)t * p.q.sT) + (long)h * p.q.sH + g4 * 16;
#pragma unroll
        for (int hf = 0; hf < HALF; ++hf)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int u = 0; u < (int)sizeof(T) / 2; ++u) {
                    q_raw[i][hf][s][u] = make_uint4(0, 0, 0, 0);
                    if (row < n_rows) q_raw[i][hf][s][u] = *(const uint4*)(from + hf * 64 + s * 8 + u * 4);
                }
    }
    auto make_q = [&]() {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint4* w = q_raw[i][hf][s];
                    if constexpr (NQ == 1) {
                        const unsigned flip = p.neg | p.neg >> 16;
                        qf[i][hf][s][0] = __builtin_bit_cast(bf16x8, make_uint4(w[0].x ^ flip, w[0].y ^ flip, w[0].z ^ flip, w[0].w ^ flip));
                    } else {
                        const unsigned u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(u[e] ^ p.neg);
                        planes<NQ, DOT>(x, qf[i][hf][s]);
                    }
                }
    };

    f32x4 o[RT][D / 16];
    float m[RT], l[RT], ms[RT];        // o holds weights * 2^-m, l weights * 2^-ms without the V scales (all in powers of two)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = ms[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[i][d] = f32x4{0, 0, 0, 0};
    }

    // blocks of 64 keys of this item, dealt to the waves
    const int blocks = min((lim_max >> 6) + ((lim_max & 63) ? 1 : 0), p.max_blocks);
    const int blk0 = split * chunk, blk1 = splits > 1 ? min(blocks, blk0 + chunk) : blocks;
    // as far as the wave that sees most
    const int tile_end = min((tile + 1) * WR * ROWS, n_rows), most = tile_end > 0 ? seen(tile_end - 1) : 0;
    const int last = __builtin_amdgcn_readfirstlane(SHARE ? most : min(lim_max, blk1 << 6));      // keys from here on are nobody's
    const int k_group = 16 * (rr >> 2), k_in = rr & 3;     // 16-key group and place in it of this lane's K rows
    int blk = blk0 + wk;

    // 64 pages from the one of block `blk` on, one to a lane: where its codes begin, its K scale and the logarithm of its V scale, so that a
    // step asks memory for nothing but codes and multiplies no addresses.  Entries behind the last key are not looked up.  In the place of a
    // page that does not exist page 0 is read, with NaN scales and its V codes taken as 0: whatever they are, rows that see none of its keys
    // keep their result.
    // A block of zeros (scale 0) has codes of zero, any scale does for the product; the smallest there is keeps it from raising the reference m
    // over the blocks that make the result.  (The rounding of log2(vs) adds |log2 vs| 2^-24 to a weight.)
    int win = 0, w_lo = 0, w_hi = 0;
    float w_ks = 0.f, w_lv = 0.f;
    int clean = 0;           // up to here the window's V scales are numbers
    auto window = [&](int from) {
        win = (from << 6) >> c.log2P;
        const bool wanted = win + lane <= (last - 1) >> c.log2P;
        const int id = wanted ? kv8_page(c, b, (long)win + lane) : -1;
        const long at = (long)max(id, 0) * c.Hkv + kvh, off = at * c.P * D;
        w_lo = (int)off;
        w_hi = (int)(off >> 32);
        w_ks = w_lv = __uint_as_float(0x7fc00000u);
        if (id >= 0) {
            const float vs = c.vs[at];
            w_ks = c.ks[at] * p.scale2;
            w_lv = __builtin_amdgcn_logf(vs == 0.f ? 0x1p-126f : vs);
        }
        const unsigned long long odd = __ballot(wanted && w_lv != w_lv);
        clean = odd ? min(last, (win + __ffsll((long long)odd) - 1) << c.log2P) : last;
    };
    // whether the pages of block x are in it
    auto in_window = [&](int x) { return (((x << 6) + 48) >> c.log2P) - win < 64; };
    // lane of the window that holds key j's page
    auto at_key = [&](int j) { return (j >> c.log2P) - win; };
    auto page_at = [&](int j) {
        const int w = at_key(j);
        return (long)((unsigned long)(unsigned)__shfl(w_lo, w, 64) | (unsigned long)(unsigned)__shfl(w_hi, w, 64) << 32);
    };
    const bool whole = c.P >= 64;                          // a block lies in one page: K and V lanes look up the same
    const int v_row = (SHARE ? wr * 16 + rr : rr) * c.P, k_row = (SHARE ? 4 * wr + k_in : k_in) * D + g4 * 16;

    uint4 kf[4][HALF], vf[D / 16];
    // where a lane's K and V of block x begin
    auto find = [&](int x, const uint8_t*& kp, const uint8_t*& vp) {
        const int jk = (x << 6) + k_group, jv = (x << 6) + 16 * g4;
        const long pk = page_at(jk), pv = whole ? pk : page_at(jv);
        kp = c.k + pk + ((jk & (c.P - 1)) * D + k_row);
        vp = c.v + pv + ((jv & (c.P - 1)) + v_row);
    };
    auto load_k = [&](const uint8_t* kp) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf) kf[t][hf] = ld_codes<(WR == 1)>(kp + t * 4 * D + hf * 64);
    };
    auto load_v = [&](const uint8_t* vp) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) vf[d] = ld_codes<(WR == 1)>(vp + d * 16 * c.P);
    };
    // SHARE: this wave's quarter of a block -- K tile wr, every fourth V tile from wr on
    bf16x8* const ops = (bf16x8*)lds;                  // [2 buffers][BUFFER / 2 of K, then as many of V]
    uint4 raw[2 * HALF];
    auto bring = [&](int x) {
        const uint8_t *kp, *vp;
        find(x, kp, vp);
#pragma unroll
        for (int hf = 0; hf < HALF; ++hf) {
            raw[hf] = ld_codes<false>(kp + hf * 64);
            raw[HALF + hf] = ld_codes<false>(vp + hf * 64 * c.P);
        }
    };
    auto convert = [&](int x) {
        const int to = (x & 1) * BUFFER + lane;
        if (clean - (x << 6) < 64) {      // leftovers may hold NaN, which a weight of 0 does not silence
            const int j = (x << 6) + 16 * g4;
            const float lv = __shfl(w_lv, at_key(j), 64);
            const int keep = lv != lv ? 0 : max(0, min(16, last - j));
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf) raw[HALF + hf] = first_bytes(raw[HALF + hf], keep);
        }
#pragma unroll
        for (int hf = 0; hf < HALF; ++hf) {
            ops[to + ((wr * HALF + hf) * 2) * 64] = codes8<F>(raw[hf].x, raw[hf].y);
            ops[to + ((wr * HALF + hf) * 2 + 1) * 64] = codes8<F>(raw[hf].z, raw[hf].w);
            ops[to + BUFFER / 2 + ((hf * 4 + wr) * 2) * 64] = codes8<F>(raw[HALF + hf].x, raw[HALF + hf].y);
            ops[to + BUFFER / 2 + ((hf * 4 + wr) * 2 + 1) * 64] = codes8<F>(raw[HALF + hf].z, raw[HALF + hf].w);
        }
    };
    if (!SHARE && blk < blk1) {
        window(blk);
        const uint8_t *kp, *vp;
        find(blk, kp, vp);
        load_k(kp);
        load_v(vp);
    }
    make_q();
    // one step; MASK: some row does not see all 64 keys, or some of them have no page
    auto step = [&](auto masked) __attribute__((always_inline)) {
        constexpr bool mask = decltype(masked)::value;
        const int j0 = blk << 6, jv = j0 + 16 * g4;
        const bool more = !SHARE && blk + WK < blk1;
        const float kscale = __shfl(w_ks, at_key(jv), 64), lv = __shfl(w_lv, at_key(jv), 64);
        const uint8_t *k_next = nullptr, *v_next = nullptr;
        if (more) {
            if (!in_window(blk + WK)) window(blk + WK);
            find(blk + WK, k_next, v_next);
        }
        const int from = (blk & 1) * BUFFER + lane;      // SHARE

        f32x4 st[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) st[i][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int hf = 0; hf < HALF; ++hf) {
                bf16x8 a0, a1;
                if constexpr (SHARE) {
                    a0 = ops[from + ((t * HALF + hf) * 2) * 64];
                    a1 = ops[from + ((t * HALF + hf) * 2 + 1) * 64];
                } else {
                    a0 = codes8<F>(kf[t][hf].x, kf[t][hf].y);
                    a1 = codes8<F>(kf[t][hf].z, kf[t][hf].w);
                }
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int pl = NQ - 1; pl >= 0; --pl) {
                        st[i][t] = mfma(a0, qf[i][hf][0][pl], st[i][t]);
                        st[i][t] = mfma(a1, qf[i][hf][1][pl], st[i][t]);
                    }
            }
        if constexpr (!SHARE) {
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_k(k_next);          // in flight under the softmax and P.V
            __builtin_amdgcn_sched_barrier(0);
        }

        bf16x8 pf[RT][2][NW];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int left = lim[i] - jv;          // keys of this lane's 16 that the row sees
            if constexpr (mask) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * t + e >= left) st[i][t][e] = -INFINITY;
            }
            if (STEP && scores && rr == 0) {
#pragma unroll
                for (int t = 0; t < 4; ++t) *(f32x4*)(scores + jv + 4 * t) = st[i][t] * kscale;
            }
            float x[16], sum, unit, lw = lv;
            auto weigh = [&](float base, float base_s) {
                // a V scale below 2^-64 of what the references stand for is taken as that: its weights would run out of exponent, and l
                // lose them
                const float least = (base - base_s) - 64.f;
                lw = lv < least ? least : lv;                     // (a NaN stays)
                const float nb = lw - base;
                unit = __builtin_amdgcn_exp2f((base - base_s) - lw);      // what the sum of x counts in l
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = __builtin_amdgcn_exp2f(fmaf(st[i][k >> 2][k & 3], kscale, nb));
                if constexpr (mask) {                            // a scale behind the end may be NaN
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k >= left) x[k] = 0.f;
                }
                sum = x[0];
#pragma unroll
                for (int k = 1; k < 16; ++k) sum += x[k];
            };
            // The references need not be the largest so far, only near it: they move when a lane's 16 weights add up to more than 2^10 (at
            // the first block they are -inf, the sum +inf), so that most blocks look for no maximum and rescale nothing.
            bool follow = true;
            if constexpr (!mask) {
                weigh(m[i], ms[i]);
                follow = __any(sum > 0x1p10f || sum * unit > 0x1p30f);
            }
            if (follow) {
                if constexpr (!mask) asm volatile("");           // rare: nothing of it belongs in front of the branch
                float mx = fmaxf(st[i][0][0], st[i][0][1]);
#pragma unroll
                for (int k = 2; k < 16; k += 2) mx = fmaxf(fmaxf(mx, st[i][k >> 2][k & 3]), st[i][k >> 2][(k & 3) + 1]);
                mx *= kscale;
                if (mask && left <= 0) mx = -INFINITY;      // nothing of these 16 keys is seen, and the scale may be any leftover
                const float mn = fmaxf(m[i], across_groups_max(mx + lv)), msn = fmaxf(ms[i], across_groups_max(mx));
                const float base = mn == -INFINITY ? 0.f : mn, base_s = msn == -INFINITY ? 0.f : msn;
                const float alpha = __builtin_amdgcn_exp2f(m[i] - base);
                l[i] *= __builtin_amdgcn_exp2f(ms[i] - base_s);
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[i][d] *= alpha;
                m[i] = mn;
                ms[i] = msn;
                weigh(base, base_s);
            }
            // (a poisoned scale of a block that is seen shows in the sum)
            if (!mask || left > 0) l[i] = fmaf(sum, unit, l[i]);
            if (lw > lv) {
                const float down = __builtin_amdgcn_exp2f(lv - lw);
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] *= down;
            }
            planes<NW, DOT>(x, pf[i][0]);
            planes<NW, DOT>(x + 8, pf[i][1]);
        }
        if constexpr (mask && !SHARE) {      // leftovers may hold NaN, which a weight of 0 does not silence
            const int keep = lv != lv ? 0 : max(0, min(16, last - jv));
#pragma unroll
            for (int d = 0; d < D / 16; ++d) vf[d] = first_bytes(vf[d], keep);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            bf16x8 a0, a1;
            if constexpr (SHARE) {
                a0 = ops[from + BUFFER / 2 + (d * 2) * 64];
                a1 = ops[from + BUFFER / 2 + (d * 2 + 1) * 64];
            } else {
                a0 = codes8<F>(vf[d].x, vf[d].y);
                a1 = codes8<F>(vf[d].z, vf[d].w);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int pl = NW - 1; pl >= 0; --pl) {
                    o[i][d] = mfma(a0, pf[i][0][pl], o[i][d]);
                    o[i][d] = mfma(a1, pf[i][1][pl], o[i][d]);
                }
        }
        if constexpr (!SHARE) {
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_v(v_next);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto steps = [&](int end) {
        for (; blk < end; blk += WK) {
            if ((SHARE ? lim_min : min(lim_min, clean)) - (blk << 6) < 64) step(std::true_type{});
            else step(std::false_type{});
        }
    };
    if constexpr (!SHARE) {
        steps(blk1);
    } else {
        const int end = min((most >> 6) + ((most & 63) ? 1 : 0), p.max_blocks);
        if (end > 0) {
            window(0);
            bring(0);
            convert(0);
            if (end > 1) bring(1);
        }
        for (blk = 0; blk < end;) {
            // this wave's pieces of block blk are in LDS, then everybody's; whoever is here is done with block blk - 1, whose buffer is
            // written next
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (blk + 1 < end) {
                convert(blk + 1);
                if (blk + 2 < end) {
                    if (!in_window(blk + 2)) window(blk);
                    bring(blk + 2);
                }
            }
            if (blk < blk1) steps(blk + 1);
            else ++blk;
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        l[i] += __shfl_xor(l[i], 16, 64);
        l[i] += __shfl_xor(l[i], 32, 64);
    }

    // join the waves that shared the keys
    if constexpr (WK > 1) {
        const int R = p.lds_rows;
        RowState* sr = (RowState*)lds;                                    // [WK][R]
        float* so = lds + WK * R * 3;                                     // [WK][R][D]
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = 16 * i + rr;
            if (r >= R) continue;
            if (g4 == 0) sr[wk * R + r] = RowState{m[i], l[i], ms[i]};
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                float* at = so + ((long)wk * R + r) * D + d * 16 + g4 * 4;
                at[0] = o[i][d][0]; at[1] = o[i][d][1]; at[2] = o[i][d][2]; at[3] = o[i][d][3];
            }
        }
        __syncthreads();
        for (int e = (wk * 64 + lane) * 4; e < (row_end - row0) * D; e += 64 * WK * 4) {
            const int r = e / D, d = e % D;
            // lane w of every eight (four) weighs wave w's part of the row: sixteen lanes or more have a row
            const RowState x = sr[(lane & (WK - 1)) * R + r];
            RowState a;
            auto larger = [](float p, float q) { return fmaxf(p, q); };
            a.m = across_waves<WK>(x.m, larger);
            a.ms = across_waves<WK>(x.ms, larger);
            // a wave without a finite score has a sum of 0, or NaN where it met a NaN
            a.l = across_waves<WK>(x.l * (x.ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.ms - a.ms)), [](float p, float q) { return p + q; });
            const float f = x.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.m - a.m);
            f32x4 acc = {0, 0, 0, 0};
            auto add = [&](auto w) {
                const float fw = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(f), 0x150 + w.value, 0xf, 0xf, true));   // lane w of the sixteen
                const float* y = so + ((long)w.value * R + r) * D + d;
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = fmaf(y[k], fw, acc[k]);
            };
            add(std::integral_constant<int, 0>{});
            add(std::integral_constant<int, 1>{});
            add(std::integral_constant<int, 2>{});
            add(std::integral_constant<int, 3>{});
            if constexpr (WK == 8) {
                add(std::integral_constant<int, 4>{});
                add(std::integral_constant<int, 5>{});
                add(std::integral_constant<int, 6>{});
                add(std::integral_constant<int, 7>{});
            }
            if constexpr (STEP) {
                float f0, f1, lse;
                result_of(a, f0, f1, lse);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float v = acc[k] * f0 * f1;
                    const T hi = from_f32<T>(v);
                    const long at = frag_elem_offset<T>(b, kvh * 64 + d + k, p.step.d);
                    ((T*)p.o.data)[at] = hi;
                    if (p.step.out_lo) ((T*)p.step.out_lo)[at] = from_f32<T>(v - to_f32<T>(hi));
                }
            } else {
                store_row<T, D>(p, b, t_first, kvh, row0 + r, d, split, splits, a, acc);
            }
        }
        if (STEP && row_out) {
            float ms0 = -INFINITY, l0 = 0.f;
            for (int w = 0; w < WK; ++w) ms0 = fmaxf(ms0, sr[w].ms);
            for (int w = 0; w < WK; ++w) l0 += sr[w].l * (sr[w].ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sr[w].ms - ms0));
            const float inv = 1.0f / l0;
            for (int j = tid; j < p.step.S; j += 64 * WK) row_out[j] = j < len ? __builtin_amdgcn_exp2f(scores[j] - ms0) * inv : 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = row0 + 16 * i + rr;
            if (row < n_rows)
#pragma unroll
                for (int d = 0; d < D / 16; ++d) store_row<T, D>(p, b, t_first, kvh, row, d * 16 + g4 * 4, split, splits, RowState{m[i], l[i], ms[i]}, o[i][d]);
        }
    }
}

// joins the parts of a row whose keys were cut: a wave per (token, head), bound by the latency of lengths, references and parts one behind
// the other (1280 rows of 128 channels 4.8 us)
template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(AttnArgs p, int tile_rows)
{
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6), row = w / p.H;
    const int h = (int)(w % p.H);
    if (row >= p.ts.N) return;
    int b = 0;
    long oat = row * p.o.sT;
    if (p.ts.tok_start) {
        // the last sequence that begins at or before the row (those behind it are empty or later)
        int n = 0;
        for (int i = lane; i < p.ts.B; i += 64) n += p.ts.tok_start[i] <= row ? 1 : 0;
        b = __builtin_amdgcn_readlane(wave_scan(n), 63) - 1;
        if (b < 0 || row >= p.ts.tok_start[b] + (long)p.ts.count(b)) return;
    } else {
        b = (int)(row / p.ts.T);
        oat = (long)b * p.o.sB + row % p.ts.T * p.o.sT;
    }
    const int splits = splits_of(p, b, chunk_of(p, tile_rows));
    if (splits == 1) return;                         // its workgroup wrote the result
    const float* part = p.part + w * p.n_split * (D + 4);
    RowState a = {-INFINITY, 0.f, -INFINITY};
    float acc[D / 64] = {};
    for (int s = lane; s < splits; s += 64) {
        a.m = fmaxf(a.m, part[s * (D + 4) + D]);
        a.ms = fmaxf(a.ms, part[s * (D + 4) + D + 2]);
    }
    auto larger = [](unsigned x, unsigned y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); };
    a.m = __uint_as_float(across_wave(__float_as_uint(a.m), larger));
    a.ms = __uint_as_float(across_wave(__float_as_uint(a.ms), larger));
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float* x = part + s * (D + 4);
        const RowState o = {x[D], x[D + 1], x[D + 2]};
        a.l += o.l * (o.ms == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(o.ms - a.ms));
        const float f = o.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(o.m - a.m);
#pragma unroll
        for (int k = 0; k < D / 64; ++k) acc[k] += x[k * 64 + lane] * f;
    }
    float f0, f1, lse;
    result_of(a, f0, f1, lse);
#pragma unroll
    for (int k = 0; k < D / 64; ++k) ((T*)p.o.data)[oat + (long)h * p.o.sH + k * 64 + lane] = from_f32<T>(acc[k] * f0 * f1);
    if (p.lse && lane == 0) p.lse[row * p.H + h] = lse;
}

// ---- host side --------------------------------------------------------------------------------------
int check_attention(const char* fn, const uw_kv8_attention_args* a)
{
    UW_REQUIRE(a, "%s: null arguments", fn);
    RUN(check_cache(fn, &a->cache));
    RUN(check_seqs(fn, &a->seqs));
    RUN(check_tokens(fn, "q", &a->q, &a->seqs));
    RUN(check_tokens(fn, "o", &a->o, &a->seqs));
    UW_REQUIRE(fabsf(a->scale) < INFINITY, "%s: scale must be a finite number", fn);
    UW_REQUIRE(a->n_heads > 0 && a->n_heads % a->cache.n_kv_heads == 0, "%s: %d query heads over %d kv heads", fn, a->n_heads, a->cache.n_kv_heads);
    return UW_OK;
}

// row tiles of 16 that a wave's registers hold: f32 keeps three planes of its queries, which 128 channels leave room for once
constexpr int max_row_tiles(size_t elem, int D) { return elem == 4 && D == 128 ? 1 : 2; }

struct AttnPlan {
    int rt, wk, wr;      // row tiles of 16 per wave, waves sharing keys, waves side by side on rows
    int n_split, target, min_chunk, tiles, max_blocks, lds_rows;
    long groups, ws_bytes;   // items of a head
};

// How a call is cut.  (Device times in us of random int8 caches, calls back to back in a graph.)
//  - up to 16 rows of a kv head: one row tile, the waves share the keys
//  - more: four waves of rows side by side (128 rows, f32 with 128 channels 64), where that gives 384 workgroups, with 128 channels 256;
//    else tiles of 16 or 32 rows whose four waves share the keys -- more workgroups for the same rows, each converting the codes for itself.
//    Measured (side by side / tiles of 32 / tiles of 16; workgroups of the first):
//      bf16  64 channels  170 rows over 1500 keys        128: 40 / 22.6 / 21.1   256: 40 / 30.9 / 35.5   384: 54 / 47 / 54   448: 54 / 56 / 64
//                                                        512: 55 / 61 / 76
//                         2048 causal rows over 4096     256: 97 / 67 / 82   384: 103 / 94 / 118   448: 106 / 111 / 144   512: 109 / 120 / 155
//                         33380 causal rows of 4 heads over 5000   190 / 257 / 325
//           128 channels  2048 causal rows over 8192     128: 254 / 122 / 166   256: 255 / 227 / 344   320: 309 / 323 / 546   384: 318 / 361 / 605
//                         170 rows over 1500             256: 55 / 54 / 80   320: 76 / 74 / 100   384: 76 / 90 / 131
//      f32   64 channels  170 rows over 1500             128: 48 / 28.2 / 24.7   384: 74 / 63 / 67   448: 75 / 75.5 / 81   512: 76 / 81 / 96
//                         2048 causal rows over 4096     256: 122 / 84 / 95   384: 146 / 124 / 142   448: 150 / 151 / 183
//           128 channels  2048 causal rows over 4096     256: 124 / - / 92   320: 135 / - / 129   384: 137 / - / 145   448: 138 / - / 197
//                         170 rows over 1500             240: 52 / - / 56   336: 68 / - / 79
//    Where the sides cross depends on how full the last tile of a head is and on how long the keys are: of 191 calls drawn at random (160 to
//    660 workgroups, 64 to 3000 tokens, up to 8000 keys) side by side is the faster one from 264 workgroups on in some and from 620 in others.
//    These bounds lose 1.8 % against the better side on average (bf16, 64 channels; 320: 3.3, 448: 2.3, 512: 4.1), 3.5 % (bf16, 128; 192: 2.6,
//    320: 3.8, 384: 8.1), 5.1 % (f32, 64; 320: 7.0, 448: 4.8) and 3.6 % (f32, 128; 192: 0.8, 320: 3.6, 384: 8.1).
//    Tiles of 16 where 64-channel rows are few, 12800 of all heads, f32 25600: 2720 rows over 1500 keys 10.6 / 14.9 (32 rows), 10880 21.1 /
//    22.6, 16320 30.2 / 28.8; f32 10880 24.7 / 28.2, 19040 36.8 / 39.0, 27200 52 / 51, 32640 67 / 63.  (Rows of 128 channels make too little
//    of a key's many bytes.)
//  - long sequences are cut further where the waves share the keys, into items of equal size (chunk_of), joined by a second launch.
//    Short ones are not: up to 32 blocks (33 where the table's last one is counted) eight waves are through as soon as a second launch is --
//    one token of 8 heads over 2048 keys 11.1 either way, over 2300 12.1 uncut and 11.4 cut, over 4000 18.1 and 11.7.  Nor are many: 512
//    tables of up to 64 blocks (2300 keys 25.6 uncut, 29.2 cut; 4000 43 and 46; ragged to 4000 33 and 37), or 4096 of any length (over 2300 183
//    and 189, over 4500 358 and 363, ragged to 8000 655 and 660).  Between these bounds the cut is worth most where the lengths are long and
//    few, and costs up to a quarter where workgroups are many already (256 over 4000 keys: 23 uncut, 30 cut).
//    At least half of the 512 items wanted are cut pieces, however many tiles there are: a quarter, half, three quarters, all: five tokens of 8
//    kv heads of 128 channels over 8 x 32768 keys 109 / 108 / 108 / 100, 60 x 8 over 8192 165 / 162 / 162 / 247.
//  - eight waves instead of four for up to 256 workgroups that are not cut: over 1500 keys 6 workgroups 10.6 / 11.5, f32 11.6 / 12.5; 256 11.6 /
//    13.2, f32 12.9 / 14.2; 320 16.9 / 16.7, f32 22.0 / 18.6; 1024 33.8 / 33.6, f32 45 / 35
//  The bounds on blocks go by the table's width, for lengths are known on the device only: under a table for 32768 tokens one window of 6 heads
//  takes 11.5 instead of 9.7, 32 ragged sequences of up to 448 tokens 10.6 instead of 7.2.
AttnPlan plan_attention(const uw_kv8_attention_args* a)
{
    AttnPlan p;
    const uw_kv8_cache* c = &a->cache;
    const int G = a->n_heads / c->n_kv_heads, B = a->seqs.B, T = a->seqs.tok_start ? 0 : a->seqs.T;
    const int64_t n_tok = a->seqs.n_tok;
    const long rows = T > 0 ? (long)T * G : (long)ceil_div(n_tok, B) * G;     // per sequence; packed: on average
    p.max_blocks = (int)std::min((long)ceil_div((long)a->seqs.table_width * c->page, 64) + 1, (1l << 25) - 1);
    p.rt = rows <= 16 ? 1 : max_row_tiles(a->seqs.dtype == UW_DTYPE_F32 ? 4 : 2, c->head_dim);
    p.wk = 4;
    p.wr = 1;
    if (rows > 32) {
        const long heads = (long)B * c->n_kv_heads;
        if (ceil_div(rows, 64 * p.rt) * heads >= (c->head_dim == 64 ? 384 : 256)) {
            p.wk = 1;
            p.wr = 4;
        } else if (c->head_dim == 64 && rows * heads < (a->seqs.dtype == UW_DTYPE_F32 ? 25600 : 12800)) {
            p.rt = 1;
        }
    }
    const int per = 16 * p.rt * p.wr;
    p.tiles = T > 0 ? ceil_div(rows, per) : 0;
    p.groups = T > 0 ? (long)B * p.tiles : n_tok * G / per + std::min((long)B, (long)n_tok);
    const long alone = p.groups * c->n_kv_heads;             // workgroups without a cut
    p.n_split = 1;
    p.target = p.min_chunk = 0;
    if (p.wk == 4 && p.max_blocks > 33 && !(alone >= 512 && p.max_blocks <= 65) && alone < 4096) {
        p.min_chunk = 8;
        // a tile's last item is a short one: they are counted in, so that all items find a place at once
        const long items = ceil_div(512, c->n_kv_heads);
        p.target = (int)std::max(std::max(items - p.groups, items / 2), 1l);
        // what one tile can be cut into: a chunk is at least the tiles' blocks over `target`
        p.n_split = std::min(T > 0 ? ceil_div(p.target, p.tiles) : p.target, ceil_div(p.max_blocks, p.min_chunk));
        // and what 256 MB of parts hold
        const int hold = (int)std::max((int64_t)1, (int64_t)(256 << 20) / (n_tok * a->n_heads * (c->head_dim + 4) * 4));
        if (hold < p.n_split) {
            p.n_split = hold;
            p.min_chunk = std::max(p.min_chunk, ceil_div(p.max_blocks, hold));
        }
        if (p.n_split > 1) p.groups += p.target;
    }
    p.lds_rows = T > 0 ? (int)std::min((long)16 * p.rt, rows) : 16 * p.rt;
    if (p.wk == 4 && p.rt == 1 && p.n_split == 1 && alone <= 256) p.wk = 8;       // few workgroups: more waves in each
    p.ws_bytes = p.n_split > 1 ? n_tok * a->n_heads * (int64_t)p.n_split * (c->head_dim + 4) * 4 : 0;
    return p;
}

template <int F, typename T, int D, int RT, int WK, int WR, bool STEP = false> int launch_attention_as(const AttnArgs& a, const AttnPlan& p, hipStream_t s)
{
    size_t lds = WR == 4 ? (size_t)2 * 64 * D * 4 : WK > 1 ? (size_t)WK * p.lds_rows * (D + 3) * 4 : 0;
    if (STEP && a.step.rows) lds += (size_t)p.max_blocks * 64 * 4;
    if (lds > 64 * 1024) {
        static PerDeviceFlag flag;
        if (flag.pending()) {
            UW_HIP_CHECK(hipFuncSetAttribute((const void*)kv8_attention_kernel<F, T, D, RT, WK, WR, STEP>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
            flag.mark();
        }
    }
    hipLaunchKernelGGL((kv8_attention_kernel<F, T, D, RT, WK, WR, STEP>), dim3((unsigned)(p.groups * a.c.Hkv)), dim3(64 * WK * WR), lds, s, a);
    UW_LAUNCH_CHECK();
    return UW_OK;
}

template <int F, typename T, int D> int launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t s)
{
    constexpr int RT = max_row_tiles(sizeof(T), D);
    if (p.wr == 4) return launch_attention_as<F, T, D, RT, 1, 4>(a, p, s);
    if (p.wk == 8) return launch_attention_as<F, T, D, 1, 8, 1>(a, p, s);
    if (p.rt == 1) RUN((launch_attention_as<F, T, D, 1, 4, 1>(a, p, s)));
    if constexpr (RT > 1) {
        if (p.rt == RT) RUN((launch_attention_as<F, T, D, RT, 4, 1>(a, p, s)));
    }
    if (p.n_split == 1) return UW_OK;
    hipLaunchKernelGGL((kv8_join_kernel<T, D>), dim3(ceil_div(a.ts.N * a.H, 4)), dim3(256), 0, s, a, 16 * p.rt);
    UW_LAUNCH_CHECK();
    return UW_OK;
}

template <int F, typename T> int launch_step(const AttnArgs& a, const AttnPlan& p, hipStream_t s)
{
    // few (window, head) pairs: more waves in each workgroup, as plan_attention has it
    return p.groups * a.c.Hkv <= 256 ? launch_attention_as<F, T, 64, 1, 8, 1, true>(a, p, s) : launch_attention_as<F, T, 64, 1, 4, 1, true>(a, p, s);
}

}  // namespace

int uw_kv8_cross_decode(int dtype, const Kv8StepParams& p, hipStream_t s)
{
    RUN(check_cache("kv8_cross_decode", p.cache));
    UW_REQUIRE(p.cache->head_dim == 64 && p.cache->n_kv_heads <= 32 && p.B > 0 && p.q && p.out && p.table && p.len && p.width > 0, "kv8_cross_decode: bad arguments");
    UW_REQUIRE(p.S > 0 && p.S <= 8192 && (long)p.width * p.cache->page >= p.S, "kv8_cross_decode: %d keys in %d pages", p.S, p.width);
    UW_REQUIRE(!p.rows || p.row_index, "kv8_cross_decode: rows without row_index");
    const int H = p.cache->n_kv_heads, d = H * 64;
    UW_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.out) & 15) == 0, "kv8_cross_decode: misaligned operands");
    uw_kv8_seqs seqs = {};
    seqs.table = p.table;
    seqs.table_width = p.width;
    AttnArgs a = {};
    a.c = view_of(p.cache, &seqs);
    a.ts = TokSpan{nullptr, p.B, 1, p.B};
    a.q = TokArg{(void*)p.q, d, d, 64};
    a.o = TokArg{p.out, d, d, 64};
    a.kv_len = p.len;
    a.H = H;
    a.G = 1;
    a.n_split = 1;
    a.tiles = 1;
    a.lds_rows = 1;
    a.scale2 = LOG2E;                 // queries come scaled
    a.step.active = p.active;
    a.step.out_lo = p.out_lo;
    a.step.d = d;
    bool any = false;
    for (int h = 0; h < 32; ++h) {
        a.step.slot[h] = (signed char)(h < H ? p.sel_slot[h] : -1);
        any = any || a.step.slot[h] >= 0;
    }
    a.step.rows = any ? p.rows : nullptr;
    a.step.rows_sB = p.rows_sB;
    a.step.rows_sSel = p.rows_sSel;
    a.step.row_index = p.row_index;
    a.step.n_rows = p.n_rows;
    a.step.S = p.S;
    AttnPlan pl = {};
    pl.groups = p.B;
    pl.lds_rows = 1;
    pl.max_blocks = a.max_blocks = ceil_div(p.S, 64);
    if (p.cache->format == UW_KV8_INT8) return dtype == UW_BF16 ? launch_step<UW_KV8_INT8, bf16_t>(a, pl, s) : launch_step<UW_KV8_INT8, float>(a, pl, s);
    return dtype == UW_BF16 ? launch_step<UW_KV8_E4M3, bf16_t>(a, pl, s) : launch_step<UW_KV8_E4M3, float>(a, pl, s);
}

extern "C" {

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
    UW_REQUIRE(pl.groups * a->cache.n_kv_heads < (1 << 22) && q.n_tok * a->n_heads <= 0x7fffffff, "uw_kv8_attention: too many rows");
    AttnArgs x = {};
    x.c = view_of(&a->cache, &q);
    x.ts = span_of(&q);
    x.q = arg_of(&a->q);
    x.o = arg_of(&a->o);
    x.lse = a->lse;
    x.kv_len = q.len;
    x.part = (float*)a->ws;
    x.H = a->n_heads;
    x.G = a->n_heads / a->cache.n_kv_heads;
    x.log2G = (x.G & (x.G - 1)) ? -1 : __builtin_ctz(x.G);
    x.causal = a->causal;
    x.n_split = pl.n_split;
    x.target = pl.target;
    x.min_chunk = pl.min_chunk;
    x.max_blocks = pl.max_blocks;
    x.tiles = pl.tiles;
    x.lds_rows = pl.lds_rows;
    x.scale2 = fabsf(a->scale) * LOG2E;
    x.neg = a->scale < 0.f ? 0x80000000u : 0u;
#define CALL(F, T) RUN((a->cache.head_dim == 64 ? launch_attention<F, T, 64>(x, pl, (hipStream_t)stream) : launch_attention<F, T, 128>(x, pl, (hipStream_t)stream)))
    KV8_DISPATCH(a->cache.format, q.dtype, CALL);
#undef CALL
    return UW_OK;
}

}  // extern "C"
