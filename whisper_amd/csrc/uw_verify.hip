// Verification of drafted tokens against the target model's scores (speculative decoding), from given random numbers.
//
//   p_i = softmax(target_i / T), q_i = softmax(draft_i / T);  token i stands while u_i q_i(d_i) < p_i(d_i);  at the first that does
//   not, the next token comes from max(p_i - q_i, 0), otherwise from p_n: the first index whose cumulative weight exceeds u_N sum w.
//
// Everything that decides about a token is held in 64 bits: a cumulative sum over a vocabulary of 50 000 has a border every 2e-5 on
// average, and in 32 bits (1e-7 a step) about one draw in a hundred would fall on the wrong side of one.
//
// A vocabulary row is cut into chunks of 4096 scores, 16 to a thread, and three launches follow the data: (1) maximum and sum of
// exponentials of every chunk of every row -- the one pass over all scores, bound by HBM; (2) each chunk's workgroup joins the
// rows' statistics, decides how many tokens stand, and sums the weights of its chunk of the one row that is drawn from (which is
// in L2 or the Infinity Cache by then); (3) a workgroup per sequence finds the chunk, then the token in it.  Probabilities need no
// (1), logits without a draft no (2); greedy verification needs the arg-max of (1) and then one small launch.
//
// Measured: 64 windows of nought to five tokens, both models' f32 logits (V 51865, 80 MB read): 20.6 + 13.0 + 6.9 us by kernel trace, 41 in
// a row of calls.  (1) does as much f64 arithmetic as reading, 3.9 TB/s; (2) and (3) are chains of statistics, decision, scores and sums
// with few rows left to work side by side.  One window of four tokens 3.5 + 9.0 us.  Greedy, 128 windows of four tokens, bf16 (66 MB): 15.5 +
// 4.0 us, 4.3 TB/s.  Probabilities of both models, five tokens: 64 windows (26.5 MB, no (1)) 12.8 us, one 9.5.  Chunks of 2048 scores took
// 26.4 + 14.2 + 7.7 us and greedy 24.2, of 8192 23.4 + 16.6 + 13.4 and 17.5, when these took 22.7 + 14.1 + 8.6 and 17.8.
#include "../../include/uw_hip.h"
#include "uw_common.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

constexpr int CHUNK = 4096, PER = 16;      // scores per workgroup and per thread

struct ChunkStat { double z; float mx; int arg; };         // sum of exp((x - mx) / T), maximum, its lowest index (-1: a NaN, greedy only)
struct Chosen { double rp, rq; float mp, mq; int acc, mode; };   // the rows drawn from (1 / sum, maximum); mode 0: p alone, 1: p - q, 2: p without the drafted token

struct VerifyParams {
    const void *target, *draft;
    long t_sB, t_sN, d_sB, d_sN;
    const int32_t *drafted, *n_drafted;
    const float* u;
    int B, N, V, chunks;
    double per_t, least;            // log2(e) / temperature; the difference of scores that is 2^-1000
    int probs;
    int32_t *accepted, *tokens;
    ChunkStat *t_stat, *d_stat;     // [B][N + 1][chunks], [B][N][chunks]
    double* mass;                   // [B][chunks][2]: of the residual, of p
    Chosen* chosen;                 // [B]

    __device__ __forceinline__ int n_of(int b) const { return n_drafted ? min(max(n_drafted[b], 0), N) : N; }
};

// 2^t, t = d * per_t, for -1000 <= t <= 0: 2^n 2^r with n the nearest whole number (what t + 1.5 2^52 has in its last bits), |r| <= 1/2;
// 2^r by the polynomial that meets it at the nine Chebyshev nodes of [-1/2, 1/2], 1.1e-12 off at most; n added to the exponent.  That
// moves one draw in ten million across a border between two tokens (2e-5 apart on average); the uniform numbers come in steps of 6e-8.
// Twelve f64 instructions; they are what these kernels wait for as much as for memory (with eighteen, 64 windows took 48 us, with twelve 43).
// A NaN stays one.
__device__ __forceinline__ double pow2_near(double d, double per_t)
{
    const double whole = 6755399441055744.0, s = fma(d, per_t, whole), r = fma(d, per_t, whole - s);
    double y = 1.3255199372687166e-06;
    y = fma(y, r, 1.5310079984429433e-05);
    y = fma(y, r, 0.00015403455966378488);
    y = fma(y, r, 0.0013333450565774538);
    y = fma(y, r, 0.009618129159246654);
    y = fma(y, r, 0.05550410941208298);
    y = fma(y, r, 0.24022650695813655);
    y = fma(y, r, 0.6931471805459328);
    y = fma(y, r, 1.0);
    return __hiloint2double(__double2hiint(y) + (__double2loint(s) << 20), __double2loint(y));
}
// the same for all d <= 0: 0 below 2^-1000, so that a score of -inf has no weight at all
__device__ __forceinline__ double pow2_neg(double d, const VerifyParams& p)
{
    const double y = pow2_near(d, p.per_t);
    return d < p.least ? 0.0 : y;
}

// PER scores of a chunk: piece u of thread t begins at u * 256 * VEC + t * VEC; -inf behind the row's end.  Rows begin at any address
// that a score may have, so the 16-byte loads assume no more.
template <typename T> struct Piece;
template <> struct Piece<float> { typedef float V __attribute__((ext_vector_type(4), aligned(4))); static constexpr int VEC = 4; };
template <> struct Piece<bf16_t> { typedef unsigned short V __attribute__((ext_vector_type(8), aligned(2))); static constexpr int VEC = 8; };
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(unsigned short x) { return __uint_as_float((unsigned)x << 16); }

template <typename T> __device__ __forceinline__ int score_index(int j0, int k)
{
    constexpr int VEC = Piece<T>::VEC;
    return j0 + (k / VEC) * 256 * VEC + (int)threadIdx.x * VEC + k % VEC;
}
template <typename T> __device__ __forceinline__ void load_scores(const T* row, int j0, int V, float* x, float fill)
{
    constexpr int VEC = Piece<T>::VEC;
#pragma unroll
    for (int u = 0; u < PER / VEC; ++u) {
        const int j = score_index<T>(j0, u * VEC);
        if (j + VEC <= V) {
            const typename Piece<T>::V v = *(const typename Piece<T>::V*)(row + j);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[u * VEC + e] = widen(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[u * VEC + e] = j + e < V ? to_f32<T>(row[j + e]) : fill;
        }
    }
}

// Sums and extremes over a wave or over sixteen lanes, by moves inside the vector ALU (a trip through LDS for each step would make up a
// third of the small launches).  Their order is fixed, and the same for every lane that gets the result.
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ double moved(double v)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, true),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ double lane_d(double v, int lane)
{
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
// sums of lanes 0 .. own: shifts inside the rows of sixteen, then the rows' totals handed on
__device__ __forceinline__ double wave_sums_d(double v)
{
    v += moved<0x111>(v);
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    v += moved<0x118>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double wave_sum_d(double v) { return lane_d(wave_sums_d(v), 63); }
__device__ __forceinline__ double row_sum_d(double v)
{
    v += moved<0x128>(v);
    v += moved<0x124>(v);
    v += moved<0x122>(v);
    v += moved<0x121>(v);
    return v;
}
__device__ __forceinline__ unsigned larger_f(unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
__device__ __forceinline__ float row_max_f(float x) { return __uint_as_float(across_row(__float_as_uint(x), larger_f)); }
__device__ __forceinline__ float wave_max_f(float x) { return __uint_as_float(across_wave(__float_as_uint(x), larger_f)); }
__device__ __forceinline__ int wave_min_i(int x) { return (int)across_wave((unsigned)x, [](unsigned a, unsigned b) { return (unsigned)min((int)a, (int)b); }); }
__device__ __forceinline__ int wave_max_i(int x) { return (int)across_wave((unsigned)x, [](unsigned a, unsigned b) { return (unsigned)max((int)a, (int)b); }); }

// (1) grid (chunks, B * (N + 1) target rows, then B * N draft rows)
template <typename T, bool GREEDY>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyParams p)
{
    __shared__ double s_z[4];
    __shared__ float s_m[4];
    __shared__ int s_a[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c = blockIdx.x % p.chunks;
    int row = blockIdx.x / p.chunks;
    const bool is_draft = row >= p.B * (p.N + 1);
    if (is_draft) row -= p.B * (p.N + 1);
    const int per = is_draft ? p.N : p.N + 1, b = row / per, i = row % per;
    if (i > p.n_of(b) - (is_draft ? 1 : 0)) return;                // no token there: nothing reads its statistics
    const T* x0 = is_draft ? (const T*)p.draft + (long)b * p.d_sB + (long)i * p.d_sN : (const T*)p.target + (long)b * p.t_sB + (long)i * p.t_sN;
    const int j0 = c * CHUNK;
    float x[PER];
    load_scores<T>(x0, j0, p.V, x, -INFINITY);
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) mx = fmaxf(mx, x[k]);
    mx = wave_max_f(mx);
    if (lane == 0) s_m[wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    ChunkStat* out = (is_draft ? p.d_stat : p.t_stat) + (long)row * p.chunks + c;
    if constexpr (GREEDY) {
        int arg = 0x7fffffff;
        bool bad = false;
#pragma unroll
        for (int k = PER - 1; k >= 0; --k) {
            if (x[k] == mx) arg = score_index<T>(j0, k);            // a thread's indexes ascend with k
            bad |= x[k] != x[k];
        }
        arg = wave_min_i(arg);
        if (lane == 0) s_a[wave] = arg;
        bad = __syncthreads_or(bad);
        if (tid == 0) *out = ChunkStat{0.0, mx, bad ? -1 : min(min(s_a[0], s_a[1]), min(s_a[2], s_a[3]))};
    } else {
        // (2^-1000 for what is smaller, -inf too: nothing beside the 1 of the maximum, and a chunk of -inf is not summed)
        double z = 0;
        bool bad = mx == INFINITY;
#pragma unroll
        for (int k = 0; k < PER; k += 2) bad |= (bool)__builtin_isunordered(x[k], x[k + 1]);
        if (mx != -INFINITY) {
#pragma unroll
            for (int k = 0; k < PER; ++k) z += pow2_near(fmax((double)x[k] - (double)mx, p.least), p.per_t);
        }
        z = wave_sum_d(bad ? (double)NAN : z);
        if (lane == 0) s_z[wave] = z;
        __syncthreads();
        if (tid == 0) *out = ChunkStat{(s_z[0] + s_z[1]) + (s_z[2] + s_z[3]), mx, 0};
    }
}

// maximum and sum of a whole row from its chunks, by 16 lanes, the same in all of them and -- the order being fixed -- in all workgroups
__device__ __forceinline__ void join_row(const VerifyParams& p, const ChunkStat* st, float& m, double& z)
{
    const int lane = threadIdx.x & 15;
    m = -INFINITY;
    for (int c = lane; c < p.chunks; c += 16) m = fmaxf(m, st[c].mx);
    m = row_max_f(m);
    z = 0;
    for (int c = lane; c < p.chunks; c += 16) {
        const ChunkStat s = st[c];
        z += s.mx == -INFINITY ? s.z : s.z * pow2_neg((double)s.mx - (double)m, p);    // (z of a chunk of -inf is 0, or NaN)
    }
    z = row_sum_d(z);
}

// r: 1 / sum of the row's exponentials
__device__ __forceinline__ double probability(const VerifyParams& p, float x, float m, double r)
{
    return p.probs ? (double)x : pow2_neg((double)x - (double)m, p) * r;
}

// How many of a sequence's tokens stand, and the rows that the next one is drawn from: by all 256 threads, the same in all of them.
// Eight positions at a time, 16 lanes to a row -- even slots the target's rows, odd ones the draft's -- so that all their statistics
// are on their way at once.
struct DecideScratch { double r[16], p[16]; float m[16], u[8]; };       // of a batch of rows: 1 / sum, probability of the drafted token
template <typename T> __device__ __forceinline__ Chosen decide(const VerifyParams& p, int b, DecideScratch& s)
{
    const int tid = threadIdx.x, n = p.n_of(b);
    const T* tb = (const T*)p.target + (long)b * p.t_sB;
    const T* db = p.draft ? (const T*)p.draft + (long)b * p.d_sB : nullptr;
    const int32_t* d = p.drafted + (long)b * p.N;
    int acc;
    for (int i0 = 0;; i0 += 8) {
        const int slot = tid >> 4, i = i0 + (slot >> 1);
        const bool is_draft = slot & 1;
        if (i <= n && (!is_draft || (db && i < n))) {
            const int di = i < n ? d[i] : -1;
            const bool token = di >= 0 && di < p.V;
            const float x = !token ? 0.f : is_draft ? to_f32<T>(db[(long)i * p.d_sN + di]) : to_f32<T>(tb[(long)i * p.t_sN + di]);
            float m = 0;
            double z = 1;
            if (!p.probs) {
                if (is_draft) join_row(p, p.d_stat + ((long)b * p.N + i) * p.chunks, m, z);
                else join_row(p, p.t_stat + ((long)b * (p.N + 1) + i) * p.chunks, m, z);
            }
            const double r = 1.0 / z;
            if ((tid & 15) == 0) {
                if (!is_draft) s.u[slot >> 1] = i < n ? p.u[(long)b * (p.N + 1) + i] : 0.f;
                s.m[slot] = m;
                s.r[slot] = r;
                s.p[slot] = !token ? 0.0 : probability(p, x, m, r);       // an id outside the vocabulary is never accepted
            }
        }
        __syncthreads();
        int run = 0;
        while (run < 8 && i0 + run < n && (double)s.u[run] * (db ? s.p[2 * run + 1] : 1.0) < s.p[2 * run]) ++run;
        acc = i0 + run;
        if (run < 8) break;
        __syncthreads();
    }
    const bool residual = db && acc < n, point = !db && acc < n && d[acc] >= 0 && d[acc] < p.V;
    const int at = (acc & 7) * 2;
    return Chosen{s.r[at], residual ? s.r[at + 1] : 1.0, s.m[at], residual ? s.m[at + 1] : 0.f, acc, residual ? 1 : point ? 2 : 0};
}

// (2) grid (chunks, B)
template <typename T>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyParams p)
{
    __shared__ DecideScratch scratch;
    __shared__ double s_z[4], s_w[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x % p.chunks, b = blockIdx.x / p.chunks, V = p.V;
    const Chosen ch = decide<T>(p, b, scratch);
    const T* row = (const T*)p.target + (long)b * p.t_sB + (long)ch.acc * p.t_sN;
    const T* qrow = ch.mode == 1 ? (const T*)p.draft + (long)b * p.d_sB + (long)ch.acc * p.d_sN : nullptr;
    const int point = ch.mode == 2 ? p.drafted[(long)b * p.N + ch.acc] : -1;
    float x[PER], y[PER];
    const int j0 = c * CHUNK;
    const float none = p.probs ? 0.f : -INFINITY;
    load_scores<T>(row, j0, V, x, none);
    if (qrow) load_scores<T>(qrow, j0, V, y, none);
    double sp = 0, sr = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const double w = probability(p, x[k], ch.mp, ch.rp);
        sp += w;
        if (qrow) {
            const double r = w - probability(p, y[k], ch.mq, ch.rq);
            sr += r != r ? r : fmax(r, 0.0);
        } else if (score_index<T>(j0, k) != point) {
            sr += w;
        }
    }
    sp = wave_sum_d(sp);
    sr = wave_sum_d(sr);
    if (lane == 0) { s_z[wave] = sp; s_w[wave] = sr; }
    __syncthreads();
    if (tid == 0) {
        double* at = p.mass + ((long)b * p.chunks + c) * 2;
        at[0] = (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]);
        at[1] = (s_z[0] + s_z[1]) + (s_z[2] + s_z[3]);
        if (c == 0) p.chosen[b] = ch;
    }
}

// the answer of one sequence
__device__ __forceinline__ void write_tokens(const VerifyParams& p, int b, int acc, int next)
{
    if (threadIdx.x == 0) p.accepted[b] = acc;
    for (int i = threadIdx.x; i <= p.N; i += blockDim.x)
        p.tokens[(long)b * (p.N + 1) + i] = i < acc ? p.drafted[(long)b * p.N + i] : i == acc ? next : -1;
}

// (3) grid B: which chunk, then which token.  OWN: logits without a draft -- the chunks' sums of (1) are their masses but for the one that
// loses the drafted token, so (2) is not needed.
template <typename T, bool OWN>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyParams p)
{
    __shared__ DecideScratch scratch;
    __shared__ double s_c[8];
    __shared__ double s_r;
    __shared__ int s_chunk, s_next, s_last[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, V = p.V;
    const Chosen ch = OWN ? decide<T>(p, b, scratch) : p.chosen[b];
    const double* mass = p.mass + (long)b * p.chunks * 2;
    const ChunkStat* st = p.t_stat + ((long)b * (p.N + 1) + ch.acc) * p.chunks;
    const T* row = (const T*)p.target + (long)b * p.t_sB + (long)ch.acc * p.t_sN;
    const T* qrow = (const T*)p.draft + (long)b * p.d_sB + (long)ch.acc * p.d_sN;
    const int point = ch.mode == 2 ? p.drafted[(long)b * p.N + ch.acc] : -1;

    double without = 0;                       // OWN: mass of the drafted token's chunk without it
    if (OWN && ch.mode == 2) {
        float x[PER];
        const int j0 = point / CHUNK * CHUNK;
        load_scores<T>(row, j0, V, x, -INFINITY);
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (score_index<T>(j0, k) != point) without += probability(p, x[k], ch.mp, ch.rp);
        without = wave_sum_d(without);
        if (lane == 0) s_c[wave] = without;
        __syncthreads();
        without = (s_c[0] + s_c[1]) + (s_c[2] + s_c[3]);
        __syncthreads();
    }
    // of the residual (0) or of p (1)
    auto mass_of = [&](int c, int which) {
        if constexpr (!OWN) return mass[2 * c + which];
        if (which == 0 && ch.mode == 2 && c == point / CHUNK) return without;
        const ChunkStat s = st[c];
        return (s.mx == -INFINITY ? s.z : s.z * pow2_neg((double)s.mx - (double)ch.mp, p)) * ch.rp;
    };
    // totals: a thread a chunk, added up wave by wave in a fixed order
    double own[2] = {0, 0};
    for (int c = tid; c < p.chunks; c += 256) { own[0] += mass_of(c, 0); own[1] += mass_of(c, 1); }
    own[0] = wave_sum_d(own[0]);
    own[1] = wave_sum_d(own[1]);
    if (lane == 0) { s_c[wave] = own[0]; s_c[4 + wave] = own[1]; }
    __syncthreads();
    const double tot[2] = {(s_c[0] + s_c[1]) + (s_c[2] + s_c[3]), (s_c[4] + s_c[5]) + (s_c[6] + s_c[7])};
    // an empty residual (probabilities that do not add up alike) leaves the row itself
    const int which = (ch.mode == 0 || tot[0] == 0.0) ? 1 : 0;
    const double total = tot[which];
    if (!(total > 0.0 && total < INFINITY)) { write_tokens(p, b, ch.acc, -1); return; }
    const double r = (double)p.u[(long)b * (p.N + 1) + p.N] * total;
    // the first chunk whose cumulative weight exceeds r; if rounding leaves none, the last one with weight
    if (wave == 0) {
        double cum = 0, before = 0, last_before = 0;
        int at = -1, last = 0;
        for (int c0 = 0; c0 < p.chunks && at < 0; c0 += 64) {
            const double w = c0 + lane < p.chunks ? mass_of(c0 + lane, which) : 0.0;
            const double incl = cum + wave_sums_d(w), excl = incl - w;
            const unsigned long long some = __ballot(w > 0), over = __ballot(w > 0 && incl > r);
            if (some) {
                const int k = 63 - __clzll((long long)some);
                last = c0 + k;
                last_before = lane_d(excl, k);
            }
            if (over) {
                const int k = __ffsll((long long)over) - 1;
                at = c0 + k;
                before = lane_d(excl, k);
            }
            cum = lane_d(incl, 63);
        }
        if (lane == 0) {
            s_chunk = at < 0 ? last : at;
            s_r = r - (at < 0 ? last_before : before);
            s_next = 0x7fffffff;
        }
    }
    __syncthreads();
    const int j0 = s_chunk * CHUNK, b0 = j0 + tid * PER;
    const int mode = which ? 0 : ch.mode;
    // a thread's 16 scores follow one another here, so that its weights can be added up in order
    constexpr int VEC = Piece<T>::VEC;
    auto run_of = [&](const T* from, float* x) {
#pragma unroll
        for (int k = 0; k < PER; k += VEC) {
            if (b0 + k + VEC <= V) {
                const typename Piece<T>::V v = *(const typename Piece<T>::V*)(from + b0 + k);
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[k + e] = widen(v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[k + e] = b0 + k + e < V ? to_f32<T>(from[b0 + k + e]) : (p.probs ? 0.f : -INFINITY);
            }
        }
    };
    float x[PER], y[PER];
    run_of(row, x);
    if (mode == 1) run_of(qrow, y);
    double w[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        double v = probability(p, x[k], ch.mp, ch.rp);
        if (mode == 1) v = fmax(v - probability(p, y[k], ch.mq, ch.rq), 0.0);
        if (mode == 2 && b0 + k == point) v = 0;
        w[k] = v;
        sum += v;
    }
    double incl = wave_sums_d(sum);
    if (lane == 63) s_c[wave] = incl;
    __syncthreads();
    for (int k = 0; k < wave; ++k) incl += s_c[k];
    double cum = incl - sum;
    int found = 0x7fffffff, last = -1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        cum += w[k];
        if (w[k] > 0) last = b0 + k;
        if (w[k] > 0 && cum > s_r) found = min(found, b0 + k);
    }
    found = wave_min_i(found);
    last = wave_max_i(last);
    if (lane == 0) { s_last[wave] = last; atomicMin(&s_next, found); }      // (a minimum: the order of arrival is nothing to it)
    __syncthreads();
    const int next = s_next != 0x7fffffff ? s_next : max(max(s_last[0], s_last[1]), max(s_last[2], s_last[3]));
    write_tokens(p, b, ch.acc, next);
}

// greedy: grid B
__global__ __launch_bounds__(256) void verify_greedy_kernel(VerifyParams p)
{
    __shared__ int s_a[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.x, n = p.n_of(b);
    const ChunkStat* ts = p.t_stat + (long)b * (p.N + 1) * p.chunks;
    int acc = 0, next = -1;
    for (int i0 = 0;; i0 += 4) {
        const int i = i0 + wave;
        int arg = 0x7fffffff;
        if (i <= n) {
            float m = -INFINITY;
            bool bad = false;
            for (int c = lane; c < p.chunks; c += 64) {
                const ChunkStat s = ts[(long)i * p.chunks + c];
                bad |= s.arg < 0;
                if (s.mx > m || arg == 0x7fffffff) { m = s.mx; arg = s.arg; }      // chunks ascend: the first of equal ones stays
            }
            const float top = wave_max_f(m);
            if (m != top) arg = 0x7fffffff;
            arg = wave_min_i(arg);
            if (__any(bad)) arg = -1;
        }
        if (lane == 0) s_a[wave] = arg;
        __syncthreads();
        int w = 0;
        for (; w < 4; ++w) {
            next = s_a[w];
            acc = i0 + w;
            if (acc >= n || next < 0 || next != p.drafted[(long)b * p.N + acc]) break;
        }
        __syncthreads();
        if (w < 4) break;
    }
    write_tokens(p, b, acc, next);
}

long chunks_of(const uw_verify_args* a) { return ceil_div(a->V, CHUNK); }
bool all_rows(const uw_verify_args* a) { return !a->probs || a->temperature == 0.0; }
int64_t workspace_bytes(const uw_verify_args* a)
{
    const int64_t rows = all_rows(a) ? (int64_t)a->B * (a->N + 1 + (a->temperature > 0.0 && a->draft ? a->N : 0)) : 0;
    return rows * chunks_of(a) * (int64_t)sizeof(ChunkStat) + (int64_t)a->B * (chunks_of(a) * 16 + (int64_t)sizeof(Chosen));
}

int check_verify(const uw_verify_args* a)
{
    UW_REQUIRE(a, "uw_verify_draft: null arguments");
    UW_REQUIRE(a->dtype == UW_DTYPE_F32 || a->dtype == UW_DTYPE_BF16, "uw_verify_draft: dtype must be f32 or bf16");
    UW_REQUIRE(a->B > 0 && a->N >= 0 && a->V > 0, "uw_verify_draft: B %d, N %d, V %d", a->B, a->N, a->V);
    UW_REQUIRE(a->V <= 0x7fffffff - CHUNK && (double)a->B * (2.0 * a->N + 1) * ((a->V + CHUNK - 1) / CHUNK) < (1 << 24), "uw_verify_draft: too many rows");
    UW_REQUIRE(a->target && a->accepted && a->tokens && (a->drafted || a->N == 0), "uw_verify_draft: null argument");
    UW_REQUIRE(a->temperature >= 0.0 && a->temperature < INFINITY, "uw_verify_draft: temperature must be finite and not negative");
    UW_REQUIRE(a->uniforms || a->temperature == 0.0, "uw_verify_draft: uniforms missing");
    UW_REQUIRE(!a->probs || a->temperature == 1.0 || a->temperature == 0.0, "uw_verify_draft: probabilities take no temperature");
    UW_REQUIRE((((uintptr_t)a->target | (uintptr_t)a->draft) & (a->dtype == UW_DTYPE_F32 ? 3 : 1)) == 0, "uw_verify_draft: misaligned rows");
    return UW_OK;
}

}  // namespace

extern "C" {

int64_t uw_verify_draft_workspace_bytes(const uw_verify_args* a) { return check_verify(a) ? -1 : workspace_bytes(a); }

int uw_verify_draft(const uw_verify_args* a, void* stream)
{
    const int rc = check_verify(a);
    if (rc) return rc;
    UW_REQUIRE(a->ws && ((uintptr_t)a->ws & 15) == 0 && a->ws_bytes >= workspace_bytes(a),
               "uw_verify_draft: workspace missing, misaligned or smaller than %lld bytes", (long long)workspace_bytes(a));
    const bool greedy = a->temperature == 0.0;
    const long chunks = chunks_of(a), t_rows = (long)a->B * (a->N + 1), d_rows = !greedy && a->draft ? (long)a->B * a->N : 0;
    VerifyParams p;
    p.target = a->target;
    p.draft = greedy ? nullptr : a->draft;
    p.t_sB = a->target_sB;
    p.t_sN = a->target_sN;
    p.d_sB = a->draft_sB;
    p.d_sN = a->draft_sN;
    p.drafted = a->drafted;
    p.n_drafted = a->n_drafted;
    p.u = a->uniforms;
    p.B = a->B;
    p.N = a->N;
    p.V = a->V;
    p.chunks = (int)chunks;
    // (beyond these bounds nothing changes: from 1e-60 down any two f32 scores that differ are 2^-1000 apart, from 1e60 up none are)
    p.per_t = greedy ? 0.0 : 1.4426950408889634074 / std::min(std::max(a->temperature, 1e-60), 1e60);
    p.least = greedy ? 0.0 : -1000.0 / p.per_t;
    p.probs = a->probs;
    p.accepted = a->accepted;
    p.tokens = a->tokens;
    p.chosen = (Chosen*)a->ws;
    p.mass = (double*)(p.chosen + a->B);
    p.t_stat = (ChunkStat*)(p.mass + (long)a->B * chunks * 2);
    p.d_stat = p.t_stat + t_rows * chunks;
    const hipStream_t s = (hipStream_t)stream;
    const bool f32 = a->dtype == UW_DTYPE_F32;
    const dim3 rows((unsigned)(chunks * (t_rows + d_rows))), one(256);
    if (greedy) {
        if (f32) hipLaunchKernelGGL((verify_rows_kernel<float, true>), rows, one, 0, s, p);
        else hipLaunchKernelGGL((verify_rows_kernel<bf16_t, true>), rows, one, 0, s, p);
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(a->B), one, 0, s, p);
    } else {
        const dim3 mass((unsigned)(chunks * a->B));
        if (!a->probs) {
            if (f32) hipLaunchKernelGGL((verify_rows_kernel<float, false>), rows, one, 0, s, p);
            else hipLaunchKernelGGL((verify_rows_kernel<bf16_t, false>), rows, one, 0, s, p);
        }
        const dim3 seqs(a->B);
        if (!a->probs && !a->draft) {
            if (f32) hipLaunchKernelGGL((verify_pick_kernel<float, true>), seqs, one, 0, s, p);
            else hipLaunchKernelGGL((verify_pick_kernel<bf16_t, true>), seqs, one, 0, s, p);
        } else if (f32) {
            hipLaunchKernelGGL(verify_mass_kernel<float>, mass, one, 0, s, p);
            hipLaunchKernelGGL((verify_pick_kernel<float, false>), seqs, one, 0, s, p);
        } else {
            hipLaunchKernelGGL(verify_mass_kernel<bf16_t>, mass, one, 0, s, p);
            hipLaunchKernelGGL((verify_pick_kernel<bf16_t, false>), seqs, one, 0, s, p);
        }
    }
    UW_LAUNCH_CHECK();
    return UW_OK;
}

}  // extern "C"
