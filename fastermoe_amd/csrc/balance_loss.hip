// Balance loss of a gate with the experts' counts and mean probabilities, and its gradient (gfx950).
//
//   c_e = slots of counted tokens that name expert e     P_e = sum over counted tokens of softmax(logits)_e
//   T counted tokens, S = sum_e c_e slots                loss = E sum_e c_e P_e / D^2,  D = T or S        prob_e = P_e / T
//   u_e = grad_loss E (c_e - S / E) / D^2 + grad_prob_e / T         grad_logits[t,e] = p_te (u_e - sum_f p_tf u_f)
//
// (The gradient does not feel a constant added to u, as the probabilities of a token add up to one: with the counts less
// their mean, taken before anything is rounded, no two nearly equal numbers are subtracted where the experts are nearly balanced.)
#include "common.hpp"

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;
constexpr int kMostExperts = 8192;
constexpr int kMostParts = 256;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// The row's largest logit and the reciprocal of the sum of exp(logit - largest), by one wave.  A row of minus infinities has no
// probabilities: the reciprocal is 0, so that they come out as zeros.
struct RowTerms { float most, inv; };
template <typename T> __device__ __forceinline__ RowTerms row_terms(const T *row, int n_expert) {
    const int lane = threadIdx.x % kWave;
    float m = -INFINITY, s = 0.f;
    for (int e = lane; e < n_expert; e += kWave) m = fmaxf(m, (float)row[e]);
    m = wave_max(m);
    if (m == -INFINITY) m = 0.f;
    for (int e = lane; e < n_expert; e += kWave) s += expf((float)row[e] - m);
    s = wave_sum(s);
    return RowTerms{m, s == 0.f ? 0.f : 1.f / s};
}

template <typename T>
__global__ __launch_bounds__(kBlock) void balance_rows_kernel(const T *__restrict__ logits, const uint8_t *__restrict__ mask,
                                                              float2 *__restrict__ terms, int64_t n_tokens, int n_expert) {
    const int64_t t = (int64_t)blockIdx.x * kWavesPerBlock + threadIdx.x / kWave;
    if (t >= n_tokens) return;
    RowTerms r{0.f, 0.f};
    if (!mask || mask[t] == 0) r = row_terms(logits + t * n_expert, n_expert);
    if (threadIdx.x % kWave == 0) terms[t] = make_float2(r.most, r.inv);
}

// A range of tokens and 256 experts per workgroup, an expert to each thread
template <typename T>
__global__ __launch_bounds__(kBlock) void balance_sum_kernel(const T *__restrict__ logits, const int64_t *__restrict__ idx,
                                                             const uint8_t *__restrict__ mask, const float2 *__restrict__ terms,
                                                             float *__restrict__ part_p, int *__restrict__ part_c,
                                                             int *__restrict__ part_t, int64_t n_tokens, int n_expert, int top_k) {
    __shared__ int count[kBlock];
    const int e0 = blockIdx.x * kBlock, e = e0 + threadIdx.x;
    const int64_t per = (n_tokens + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = lo + per < n_tokens ? lo + per : n_tokens;
    count[threadIdx.x] = 0;
    __syncthreads();
    for (int64_t s = lo * top_k + threadIdx.x; s < hi * top_k; s += kBlock) {
        const int64_t named = idx[s] - e0;
        if (idx[s] >= 0 && idx[s] < n_expert && named >= 0 && named < kBlock && (!mask || mask[s / top_k] == 0))
            atomicAdd(&count[named], 1);
    }
    float p = 0.f;
    int tokens = 0;
    for (int64_t t = lo; t < hi; ++t) {
        if (mask && mask[t]) continue;
        ++tokens;
        const float2 r = terms[t];
        if (e < n_expert && r.y != 0.f) p += expf((float)logits[t * n_expert + e] - r.x) * r.y;
    }
    __syncthreads();
    if (e < n_expert) {
        part_p[(int64_t)blockIdx.y * n_expert + e] = p;
        part_c[(int64_t)blockIdx.y * n_expert + e] = count[threadIdx.x];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) part_t[blockIdx.y] = tokens;
}

// One workgroup: the sums over the ranges, what the gradient needs of them (slope [n_expert + 1]) and the loss
__global__ __launch_bounds__(kBlock) void balance_finish_kernel(const float *__restrict__ part_p, const int *__restrict__ part_c,
                                                                const int *__restrict__ part_t, int n_parts, int n_expert, int per_slot,
                                                                int64_t *__restrict__ count, float *__restrict__ prob,
                                                                float *__restrict__ slope, float *__restrict__ loss) {
    __shared__ double scratch[kBlock];
    __shared__ long long slots_lds;
    if (threadIdx.x == 0) slots_lds = 0;
    __syncthreads();
    long long tokens = 0, slots = 0;
    for (int g = 0; g < n_parts; ++g) tokens += part_t[g];
    double sum = 0;
    for (int e = threadIdx.x; e < n_expert; e += kBlock) {
        long long c = 0;
        double p = 0;
        for (int g = 0; g < n_parts; ++g) {
            c += part_c[(int64_t)g * n_expert + e];
            p += part_p[(int64_t)g * n_expert + e];
        }
        count[e] = c;
        slots += c;
        sum += p * (double)c;
        prob[e] = tokens ? (float)(p / (double)tokens) : 0.f;
    }
    scratch[threadIdx.x] = sum;
    atomicAdd((unsigned long long *)&slots_lds, (unsigned long long)slots);
    __syncthreads();
    slots = slots_lds;
    const long long per = per_slot ? slots : tokens;
    const double k = per ? (double)n_expert / ((double)per * (double)per) : 0.0;
    for (int e = threadIdx.x; e < n_expert; e += kBlock)
        slope[e] = (float)(k * ((double)count[e] - (double)slots / n_expert));
    if (threadIdx.x == 0) {
        double total = 0;
        for (int i = 0; i < kBlock; ++i) total += scratch[i];
        *loss = (float)(k * total);
        slope[n_expert] = tokens ? (float)(1.0 / (double)tokens) : 0.f;
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void balance_bwd_kernel(const T *__restrict__ logits, const uint8_t *__restrict__ mask,
                                                             const float *__restrict__ slope, const float *__restrict__ grad_loss,
                                                             const float *__restrict__ grad_prob, T *__restrict__ grad,
                                                             int64_t n_tokens, int n_expert) {
    const int64_t t = (int64_t)blockIdx.x * kWavesPerBlock + threadIdx.x / kWave;
    if (t >= n_tokens) return;
    const int lane = threadIdx.x % kWave;
    const T *row = logits + t * n_expert;
    T *out = grad + t * n_expert;
    RowTerms r{0.f, 0.f};
    if (!mask || mask[t] == 0) r = row_terms(row, n_expert);
    if (r.inv == 0.f) {
        for (int e = lane; e < n_expert; e += kWave) out[e] = (T)0.f;
        return;
    }
    const float gl = grad_loss ? *grad_loss : 0.f, per = slope[n_expert];
    auto u = [&](int e) { return gl * slope[e] + (grad_prob ? grad_prob[e] * per : 0.f); };
    float dot = 0.f;
    for (int e = lane; e < n_expert; e += kWave) dot += expf((float)row[e] - r.most) * r.inv * u(e);
    dot = wave_sum(dot);
    for (int e = lane; e < n_expert; e += kWave) out[e] = (T)(expf((float)row[e] - r.most) * r.inv * (u(e) - dot));
}

int n_parts(int64_t n_tokens) {
    const int64_t p = ceil_div(n_tokens < 1 ? 1 : n_tokens, 64);
    return (int)(p < kMostParts ? p : kMostParts);
}

int check(const char *who, int64_t n_tokens, int64_t n_expert, int dtype) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who,
                 dtype);
    FMOE_REQUIRE(n_tokens >= 0 && n_expert >= 1, "%s: bad sizes", who);
    if (n_expert > kMostExperts || n_tokens > INT32_MAX / 8)
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    return FMOE_OK;
}

template <typename F> void with_type(int dtype, F &&f) {
    if (dtype == FMOE_F32) f(float{});
    else if (dtype == FMOE_BF16) f(__bf16{});
    else f(_Float16{});
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int64_t fmoe_balance_loss_workspace_bytes(int64_t n_tokens, int64_t n_expert) {
    if (n_tokens < 0 || n_expert < 1) return 0;
    return 8 * n_tokens + (int64_t)n_parts(n_tokens) * (8 * n_expert + 4);
}

extern "C" int fmoe_balance_loss_forward(const void *logits, const int64_t *topk_idx, const void *token_mask, int64_t n_tokens,
                                         int64_t n_expert, int64_t top_k, int dtype, int per_slot, float *loss, int64_t *expert_count,
                                         float *prob, float *slope, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_balance_loss_forward";
    if (int rc = check(who, n_tokens, n_expert, dtype)) return rc;
    FMOE_REQUIRE(top_k >= 1 && top_k <= 65536, "%s: top_k=%lld", who, (long long)top_k);
    FMOE_REQUIRE(per_slot == 0 || per_slot == 1, "%s: per_slot=%d", who, per_slot);
    if (n_tokens * top_k > (int64_t)INT32_MAX) return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    FMOE_REQUIRE(loss && expert_count && prob && slope && (n_tokens == 0 || (logits && topk_idx)), "%s: NULL pointer", who);
    if (!workspace || workspace_bytes < fmoe_balance_loss_workspace_bytes(n_tokens, n_expert))
        return fail(FMOE_EWORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
                    (long long)fmoe_balance_loss_workspace_bytes(n_tokens, n_expert));
    hipStream_t st = (hipStream_t)stream;
    const int parts = n_parts(n_tokens);
    float2 *terms = (float2 *)workspace;
    float *part_p = (float *)(terms + n_tokens);
    int *part_c = (int *)(part_p + parts * n_expert), *part_t = part_c + parts * n_expert;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (n_tokens > 0)
            balance_rows_kernel<T><<<(int)ceil_div(n_tokens, kWavesPerBlock), kBlock, 0, st>>>((const T *)logits, (const uint8_t *)token_mask,
                                                                                              terms, n_tokens, (int)n_expert);
        balance_sum_kernel<T><<<dim3((int)ceil_div(n_expert, kBlock), parts), kBlock, 0, st>>>(
            (const T *)logits, topk_idx, (const uint8_t *)token_mask, terms, part_p, part_c, part_t, n_tokens, (int)n_expert, (int)top_k);
    });
    balance_finish_kernel<<<1, kBlock, 0, st>>>(part_p, part_c, part_t, parts, (int)n_expert, per_slot, expert_count, prob, slope, loss);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

extern "C" int fmoe_balance_loss_backward(const void *logits, const void *token_mask, const float *slope, const float *grad_loss,
                                          const float *grad_prob, void *grad_logits, int64_t n_tokens, int64_t n_expert, int dtype,
                                          void *stream) {
    const char *who = "fmoe_balance_loss_backward";
    if (int rc = check(who, n_tokens, n_expert, dtype)) return rc;
    if (n_tokens == 0) return FMOE_OK;
    FMOE_REQUIRE(logits && slope && grad_logits, "%s: NULL pointer", who);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        balance_bwd_kernel<T><<<(int)ceil_div(n_tokens, kWavesPerBlock), kBlock, 0, (hipStream_t)stream>>>(
            (const T *)logits, (const uint8_t *)token_mask, slope, grad_loss, grad_prob, (T *)grad_logits, n_tokens, (int)n_expert);
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
