// Verification of drafted tokens against the target model's scores (speculative decoding), from given random numbers.
//
// Everything that decides about a token is held in 64 bits: a cumulative sum over a vocabulary of 50 000 has a border every 2e-5 on
// average, and in 32 bits (1e-7 a step) about one draw in a hundred would fall on the wrong side of one.
#include "../../include/uw_hip.h"
#include "uw_common.h"
#include "uw_kernels.h"
#include <algorithm>

namespace {

struct VerifyParams {
    const void *target, *draft;
    long t_sB, t_sN, d_sB, d_sN;
    const int32_t *drafted, *n_drafted;
    const float* u;
    int B, N, V;
    double inv_t;
    int probs;
    int32_t *accepted, *tokens;
};

__device__ __forceinline__ double shfl_xor_d(double v, int o) { return __shfl_xor(v, o, 64); }

// sum / max over a 256-thread workgroup, valid in all threads; scratch: 4 doubles
__device__ __forceinline__ double block_sum_d(double v, double* s)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor_d(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}
__device__ __forceinline__ float block_max_f(float v, double* s)
{
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (float)fmax(fmax(s[0], s[1]), fmax(s[2], s[3]));
}

struct RowStat { float mx; double z; };

template <typename T> __device__ RowStat row_stat(const VerifyParams& p, const T* row, double* s)
{
    float mx = -INFINITY;
    bool bad = false;
    for (int j = threadIdx.x; j < p.V; j += 256) {
        const float x = to_f32<T>(row[j]);
        bad |= x != x;
        mx = fmaxf(mx, x);
    }
    bad = __syncthreads_or(bad);
    mx = block_max_f(mx, s);
    if (bad) mx = __uint_as_float(0x7fc00000u);
    double z = 0;
    for (int j = threadIdx.x; j < p.V; j += 256) z += exp(((double)to_f32<T>(row[j]) - (double)mx) * p.inv_t);
    return RowStat{mx, block_sum_d(z, s)};
}
template <typename T> __device__ __forceinline__ double prob(const VerifyParams& p, const T* row, int j, const RowStat& st)
{
    const double x = to_f32<T>(row[j]);
    return p.probs ? x : exp((x - (double)st.mx) * p.inv_t) / st.z;
}

// one workgroup per sequence
template <typename T>
__global__ __launch_bounds__(256) void verify_kernel(VerifyParams p)
{
    __shared__ double s[4];
    __shared__ double cum[256];
    __shared__ int s_i[4];
    const int b = blockIdx.x, tid = threadIdx.x;
    const int n = p.n_drafted ? min(max(p.n_drafted[b], 0), p.N) : p.N;
    const T* tb = (const T*)p.target + (long)b * p.t_sB;
    const T* db = p.draft ? (const T*)p.draft + (long)b * p.d_sB : nullptr;
    const int32_t* d = p.drafted + (long)b * p.N;
    const float* u = p.u + (long)b * (p.N + 1);
    int acc = 0, next = -1;
    if (p.inv_t == 0.0) {
        for (;; ++acc) {
            const T* row = tb + (long)acc * p.t_sN;
            float best = -INFINITY;
            int arg = 0x7fffffff;
            bool bad = false;
            for (int j = tid; j < p.V; j += 256) {
                const float x = to_f32<T>(row[j]);
                bad |= x != x;
                if (x > best || (x == best && j < arg)) { best = x; arg = j; }
            }
            bad = __syncthreads_or(bad);
            const float top = block_max_f(best, s);
            int cand = best == top ? arg : 0x7fffffff;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) cand = min(cand, __shfl_xor(cand, o, 64));
            if ((tid & 63) == 0) s_i[tid >> 6] = cand;
            __syncthreads();
            next = min(min(s_i[0], s_i[1]), min(s_i[2], s_i[3]));
            __syncthreads();
            if (bad) { next = -1; break; }
            if (acc >= n || d[acc] != next) break;
        }
    } else {
        RowStat ps{0.f, 1.0}, qs{0.f, 1.0};
        for (; acc <= n; ++acc) {
            const T* row = tb + (long)acc * p.t_sN;
            if (!p.probs) ps = row_stat<T>(p, row, s);
            if (acc == n) break;
            const int di = d[acc];
            if (di < 0 || di >= p.V) break;
            double qd = 1.0;
            if (db) {
                const T* qrow = db + (long)acc * p.d_sN;
                if (!p.probs) qs = row_stat<T>(p, qrow, s);
                qd = prob<T>(p, qrow, di, qs);
            }
            if (!((double)u[acc] * qd < prob<T>(p, row, di, ps))) break;
        }
        const T* row = tb + (long)acc * p.t_sN;
        const T* qrow = (db && acc < n) ? db + (long)acc * p.d_sN : nullptr;
        if (qrow && !p.probs) qs = row_stat<T>(p, qrow, s);
        const int point = (acc < n && !db) ? d[acc] : -1;
        // thread t owns a contiguous run of the vocabulary
        const int per = (p.V + 255) / 256, j0 = min(tid * per, p.V), j1 = min(j0 + per, p.V);
        bool residual = qrow || point >= 0;
        for (;;) {
            auto weight = [&](int j) {
                double w = prob<T>(p, row, j, ps);
                if (residual) {
                    if (j == point) w = 0;
                    else if (qrow) { const double dq = prob<T>(p, qrow, j, qs); w = (w != w || dq != dq) ? w + dq : fmax(w - dq, 0.0); }
                }
                return w;
            };
            double sum = 0;
            for (int j = j0; j < j1; ++j) sum += weight(j);
            __syncthreads();
            cum[tid] = sum;
            __syncthreads();
            if (tid == 0)
                for (int i = 1; i < 256; ++i) cum[i] += cum[i - 1];
            if (tid == 0) s_i[0] = -1;
            __syncthreads();
            const double total = cum[255];
            if (!(total > 0.0) && !(total != total) && residual) { residual = false; continue; }
            if (!(total > 0.0) || !(total < INFINITY)) break;
            const double r = (double)u[p.N] * total;
            const double before = tid ? cum[tid - 1] : 0.0;
            // the first thread whose cumulative weight exceeds r holds the token; rounding may leave none: then the last with mass
            const bool holds = cum[tid] > r && !(before > r);
            int found = -1, last = -1;
            double c = before;
            if (sum > 0)
                for (int j = j0; j < j1; ++j) {
                    const double w = weight(j);
                    c += w;
                    if (w > 0) last = j;
                    if (holds && found < 0 && c > r) found = j;
                }
            if (holds && found < 0) found = last;
            if (holds) s_i[0] = found;
            __syncthreads();
            next = s_i[0];
            if (next < 0) {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
                __syncthreads();
                if ((tid & 63) == 0) s_i[tid >> 6] = last;
                __syncthreads();
                next = max(max(s_i[0], s_i[1]), max(s_i[2], s_i[3]));
            }
            break;
        }
    }
    if (tid == 0) p.accepted[b] = acc;
    for (int i = tid; i <= p.N; i += 256) p.tokens[(long)b * (p.N + 1) + i] = i < acc ? d[i] : i == acc ? next : -1;
}

int check_verify(const uw_verify_args* a)
{
    UW_REQUIRE(a, "uw_verify_draft: null arguments");
    UW_REQUIRE(a->dtype == UW_DTYPE_F32 || a->dtype == UW_DTYPE_BF16, "uw_verify_draft: dtype must be f32 or bf16");
    UW_REQUIRE(a->B > 0 && a->N >= 0 && a->V > 0, "uw_verify_draft: B %d, N %d, V %d", a->B, a->N, a->V);
    UW_REQUIRE(a->target && a->accepted && a->tokens && (a->drafted || a->N == 0), "uw_verify_draft: null argument");
    UW_REQUIRE(a->temperature >= 0.f && a->temperature < INFINITY, "uw_verify_draft: temperature must be finite and not negative");
    UW_REQUIRE(a->uniforms || a->temperature == 0.f, "uw_verify_draft: uniforms missing");
    UW_REQUIRE(!a->probs || a->temperature == 1.f || a->temperature == 0.f, "uw_verify_draft: probabilities take no temperature");
    UW_REQUIRE((((uintptr_t)a->target | (uintptr_t)a->draft) & (a->dtype == UW_DTYPE_F32 ? 3 : 1)) == 0, "uw_verify_draft: misaligned rows");
    return UW_OK;
}

}  // namespace

extern "C" {

int64_t uw_verify_draft_workspace_bytes(const uw_verify_args* a) { return check_verify(a) ? -1 : 0; }

int uw_verify_draft(const uw_verify_args* a, void* stream)
{
    const int rc = check_verify(a);
    if (rc) return rc;
    const bool greedy = a->temperature == 0.f;
    VerifyParams p{a->target, greedy ? nullptr : a->draft, (long)a->target_sB, (long)a->target_sN, (long)a->draft_sB, (long)a->draft_sN,
                   a->drafted, a->n_drafted, a->uniforms, a->B, a->N, a->V, greedy ? 0.0 : 1.0 / (double)a->temperature, a->probs,
                   a->accepted, a->tokens};
    if (a->dtype == UW_DTYPE_F32) hipLaunchKernelGGL(verify_kernel<float>, dim3(a->B), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(verify_kernel<bf16_t>, dim3(a->B), dim3(256), 0, (hipStream_t)stream, p);
    UW_LAUNCH_CHECK();
    return UW_OK;
}

}  // extern "C"
