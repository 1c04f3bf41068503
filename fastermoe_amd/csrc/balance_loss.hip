// Balance loss of a gate with the experts' counts and mean probabilities, and its gradient (gfx950).
//
//   c_e = slots of counted tokens that name expert e     P_e = sum over counted tokens of softmax(logits)_e
//   T counted tokens, S = sum_e c_e slots                loss = E sum_e c_e P_e / D^2,  D = T or S        prob_e = P_e / T
//   u_e = grad_loss E (c_e - S / E) / D^2 + grad_prob_e / T         grad_logits[t,e] = p_te (u_e - sum_f p_tf u_f)
//
// (The gradient does not feel a constant added to u, as the probabilities of a token add up to one: with the counts less
// their mean, taken before anything is rounded, no two nearly equal numbers are subtracted where the experts are nearly balanced.)
//
// L lanes hold a token's logits, V vectors of 16 bytes to each (as many lanes and vectors as the experts need: held_logits), a wave 64 / L tokens;
// probabilities stay in registers between the one load and the sums over the tokens, which each lane keeps for its experts over all the tokens of its
// workgroup's range.  The logits are read once in each direction, some tokens ahead; at these sizes the chain from the first load over the sums
// to a second launch's results bounds the forward, the memory the larger backward passes (us, forward and backward):
//   32768 x 256 bf16, top-8    16.5  10.4        131072 x 64 f32, top-2    18.0  13.1 (5.1 TB/s)      8192 x 1024 f32, top-2   17.4  11.5
//   16384 x 64 f32, top-1      11.4   3.6        100000 x 60 bf16, top-2   15.2   9.7                 1000 x 16 f32, top-2      7.1   2.8
// (A pass for every token's largest logit and sum, one for the sums over the tokens and a workgroup for the results took 158 us of the first's forward,
// a token to a wave 25 of its backward.)  More than 2048 experts in float32, 32 vectors to a lane, do not fit: 528 bytes of scratch memory to a lane (1024 tokens of 8192
// experts: 55 us and 34).
#include "common.hpp"
#include "lane_elems.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kMostExperts = 8192;
constexpr int kMostParts = 256;      // workgroups of the forward, each of which leaves sums over its tokens
constexpr int kBwdBlock = 256, kBwdBlocks = 512;
constexpr int kFewRounds = 8;
constexpr int kSumCols = 16, kSumRanges = 64, kSumBlock = kSumCols * kSumRanges;
constexpr int waves_of(int v) { return v <= 2 ? 16 : v <= 8 ? 8 : 3; }   // of a workgroup of the forward
constexpr int ahead_of(int v) { return v == 1 ? 4 : v == 2 ? 2 : 1; }    // tokens in flight per lane

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// op over L adjacent lanes, the same in all of them
template <int L, typename F> __device__ __forceinline__ float over_lanes(float v, F &&op) {
    if (L > 1) v = op(v, dpp<0xb1>(v));      // quad_perm 1 0 3 2
    if (L > 2) v = op(v, dpp<0x4e>(v));      // quad_perm 2 3 0 1
    if (L > 4) v = op(v, dpp<0x141>(v));     // row_half_mirror
    if (L > 8) v = op(v, dpp<0x140>(v));     // row_mirror
    if (L == 32) v = op(v, __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(v), 0x401f)));   // the lane 16 away
    if (L == 64) {
        auto lane = [&](int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
        v = op(op(lane(0), lane(16)), op(lane(32), lane(48)));
    }
    return v;
}

// exp(x) for x <= 0 (or NaN): 2^h of the rounded h = x log2(e), and e^r = 1 + r of what that rounding took away, r = x - h ln(2) <= 1e-5 (ln(2) in two parts).
// Minus infinity leaves no difference, and r has to be a number then.  Off by two units in the last place.  (The exponential instruction of a rounded product alone is off
// by |x| / 2 such units besides; that one takes 9.7 us of the backward of 32768 x 256 bfloat16, this 10.4, the library's function 11.5.)
__device__ __forceinline__ float exp_down(float x) {
    const float h = x * 1.44269504088896341f;
    const float r = fmaf(-h, -1.90465429995776e-9f, fmaf(-h, 0.693147182464599609f, x));
    const float e = __builtin_amdgcn_exp2f(h);
    return fmaf(e, __builtin_amdgcn_fmed3f(r, -1.f, 1.f), e);
}

// A token's logits as its lanes hold them.
template <typename T, int L, int V, bool WHOLE> struct Logits {
    static constexpr int N = Vec<T>::N;
    u32x4 raw[V];
    // token t of n (WHOLE, experts in whole vectors: of the last one where there is none, and nothing looks at what comes, so that loads run ahead)
    __device__ __forceinline__ void load(const T *logits, int64_t t, int64_t n, int n_expert) {
        const int lane = threadIdx.x % L;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * L + lane) * N;
            if constexpr (WHOLE) raw[v] = *(const AnyVec *)(logits + (t < n ? t : n - 1) * n_expert + (c < n_expert ? c : 0));
            else raw[v] = load_vec<false>(logits + t * n_expert + c, t < n ? n_expert - c : 0, t * n_expert + c + N <= n * n_expert);
        }
    }
    // p <- exp(logit - largest), 0 behind the experts; returns the reciprocal of their sum, 0 for a token that is not `counted` or whose logits are all
    // minus infinity (it has no probabilities)
    __device__ __forceinline__ float softmax(float (&p)[V][N], bool counted, int n_expert) const {
        const int lane = threadIdx.x % L;
        float most = -INFINITY, sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float f[8];
            Vec<T>::unpack(raw[v], f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[v][i] = counted && (v * L + lane) * N + i < n_expert ? f[i] : -INFINITY;
                most = fmaxf(most, p[v][i]);
            }
        }
        most = over_lanes<L>(most, [](float a, float b) { return fmaxf(a, b); });
        if (most == -INFINITY) most = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[v][i] = exp_down(p[v][i] - most);
                sum += p[v][i];
            }
        sum = over_lanes<L>(sum, [](float a, float b) { return a + b; });
        return sum == 0.f ? 0.f : 1.f / sum;
    }
};

// What the forward leaves behind its sums over ranges of tokens, and what becomes of them
struct Sums {
    double *loss;       // [columns' workgroups]
    unsigned *done;     // workgroups of the columns that are through
    float *prob;        // [parts][experts]
    int *count;         // [parts][experts]
    int2 *total;        // [parts]: tokens, slots
};
struct Results { int64_t *count; float *prob, *slope, *loss; int per_slot; };

// expert e's results from its sums; returns its part of the loss, before the factor
__device__ __forceinline__ double finish_expert(const Results &r, int e, int n_expert, double p, long long c, long long tokens, long long slots) {
    const long long per = r.per_slot ? slots : tokens;
    const double k = per ? (double)n_expert / ((double)per * (double)per) : 0.0;
    r.count[e] = c;
    r.prob[e] = tokens ? (float)(p / (double)tokens) : 0.f;
    r.slope[e] = (float)(k * ((double)c - (double)slots / n_expert));
    if (e == 0) r.slope[n_expert] = tokens ? (float)(1.0 / (double)tokens) : 0.f;
    return k * p * (double)c;
}
__device__ __forceinline__ double lane_sum(double v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// A range of tokens to each workgroup: the experts' counts from the slots, then the sums of the probabilities.  A launch of one workgroup goes on
// to the results; otherwise balance_finish_kernel makes them.
template <typename T, int L, int V, bool WHOLE>
__global__ __launch_bounds__(waves_of(V) * kWave) void balance_sum_kernel(const T *__restrict__ logits, const int64_t *__restrict__ idx,
                                                                           const uint8_t *__restrict__ mask, Sums sums, Results results,
                                                                           int64_t n_tokens, int n_expert, int top_k) {
    constexpr int N = Vec<T>::N, kWaves = waves_of(V), kThreads = kWaves * kWave, kTokens = kWave / L, kAhead = ahead_of(V);
    __shared__ int counts[L * V * N];
    __shared__ float probs[kWaves][L * V * N];
    __shared__ int total[2];
    __shared__ double loss[kWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t per = (n_tokens + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * per, hi = lo + per < n_tokens ? lo + per : n_tokens;
    for (int e = threadIdx.x; e < n_expert; e += kThreads) counts[e] = 0;
    if (threadIdx.x < 2) total[threadIdx.x] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *sums.done = 0;
    __syncthreads();
    int slots = 0, tokens = 0;
    for (int64_t s = lo * top_k + threadIdx.x; s < hi * top_k; s += kThreads) {
        const int64_t e = idx[s];
        if (e >= 0 && e < n_expert && (!mask || mask[(uint32_t)s / (uint32_t)top_k] == 0)) {
            atomicAdd(&counts[e], 1);
            ++slots;
        }
    }
    float acc[V][N] = {};
    for (int64_t t0 = lo + wave * kTokens; t0 < hi; t0 += kWaves * kTokens * kAhead) {
        Logits<T, L, V, WHOLE> a[kAhead];
        bool counted[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t t = t0 + u * kWaves * kTokens + lane / L;
            a[u].load(logits, t, hi, n_expert);
            counted[u] = t < hi && (!mask || mask[t] == 0);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (t0 + u * kWaves * kTokens >= hi) break;
            float p[V][N];
            const float inv = a[u].softmax(p, counted[u], n_expert);
            tokens += __popcll(__ballot(counted[u] && lane % L == 0));
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[v][i] += p[v][i] * inv;
        }
    }
    // (a sum over the wave first: lanes that add to one address take turns, 1024 of them some 3 us)
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) slots += __shfl_xor(slots, off, kWave);
    if (lane == 0) {
        atomicAdd(&total[1], slots);
        atomicAdd(&total[0], tokens);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int off = L; off < kWave; off <<= 1) acc[v][i] += __shfl_xor(acc[v][i], off, kWave);
    if (lane < L) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) probs[wave][(v * L + lane) * N + i] = acc[v][i];
    }
    __syncthreads();
    double sum = 0;
    for (int e = threadIdx.x; e < n_expert; e += kThreads) {
        float p = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) p += probs[w][e];
        if (gridDim.x > 1) {
            sums.prob[(int64_t)blockIdx.x * n_expert + e] = p;
            sums.count[(int64_t)blockIdx.x * n_expert + e] = counts[e];
        } else {
            sum += finish_expert(results, e, n_expert, p, counts[e], total[0], total[1]);
        }
    }
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) sums.total[blockIdx.x] = make_int2(total[0], total[1]);
        return;
    }
    sum = lane_sum(sum);
    if (lane == 0) loss[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) sum += loss[w];
        *results.loss = (float)sum;
    }
}

// The results from the parts, kSumCols experts to a workgroup and the parts in kSumRanges ranges side by side; the last workgroup that is through adds
// up the loss, in the order of the experts.  (256 parts of 64 experts 6.1 us, of 16, where nobody has to be waited for, 3.6, of 256 7.2; one workgroup for
// 64 experts takes 8.2 and for 256, whose 512 KiB come from the other XCDs' writes, 25.)
__global__ __launch_bounds__(kSumBlock) void balance_finish_kernel(Sums sums, Results results, int n_parts, int n_expert) {
    constexpr int kWaves = kSumBlock / kWave;
    static_assert(kMostParts <= kSumBlock && kMostParts % kSumRanges == 0 && kSumCols < kWave, "a part's totals to a thread");
    __shared__ double prob[kWaves][kSumCols];
    __shared__ int count[kWaves][kSumCols];
    __shared__ long long total[2][kWaves];
    const int col = threadIdx.x % kSumCols, range = threadIdx.x / kSumCols, e = blockIdx.x * kSumCols + col, wave = threadIdx.x / kWave;
    const int2 mine = (int)threadIdx.x < n_parts ? sums.total[threadIdx.x] : make_int2(0, 0);
    double p = 0;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMostParts / kSumRanges; ++i) {
        const int g = range + i * kSumRanges;
        const bool in = g < n_parts && e < n_expert;
        p += in ? sums.prob[(int64_t)g * n_expert + e] : 0.f;
        c += in ? sums.count[(int64_t)g * n_expert + e] : 0;
    }
    long long tokens = mine.x, slots = mine.y;
#pragma unroll
    for (int off = kSumCols; off < kWave; off <<= 1) {
        p += __shfl_xor(p, off, kWave);
        c += __shfl_xor(c, off, kWave);
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        tokens += __shfl_xor(tokens, off, kWave);
        slots += __shfl_xor(slots, off, kWave);
    }
    if (threadIdx.x % kWave < kSumCols) {
        prob[wave][col] = p;
        count[wave][col] = c;
    }
    if (threadIdx.x % kWave == 0) {
        total[0][wave] = tokens;
        total[1][wave] = slots;
    }
    __syncthreads();
    if (wave != 0) return;
    double sum = 0;
    if (range == 0 && e < n_expert) {
#pragma unroll
        for (int r = 1; r < kWaves; ++r) {
            p += prob[r][col];
            c += count[r][col];
        }
        tokens = slots = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            tokens += total[0][w];
            slots += total[1][w];
        }
        sum = finish_expert(results, e, n_expert, p, c, tokens, slots);
    }
    sum = lane_sum(sum);
    if (gridDim.x > 1) {
        unsigned before = 0;
        if (threadIdx.x == 0) {
            __hip_atomic_store(&sums.loss[blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            before = __hip_atomic_fetch_add(sums.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (__builtin_amdgcn_readfirstlane(before) != gridDim.x - 1) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        sum = 0;
        for (unsigned i = threadIdx.x; i < gridDim.x; i += kWave) sum += __hip_atomic_load(&sums.loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sum = lane_sum(sum);
    }
    if (threadIdx.x == 0) *results.loss = (float)sum;
}

template <typename T, int L, int V, bool WHOLE, int AHEAD>
__global__ __launch_bounds__(kBwdBlock) void balance_bwd_kernel(const T *__restrict__ logits, const uint8_t *__restrict__ mask,
                                                                const float *__restrict__ slope, const float *__restrict__ grad_loss,
                                                                const float *__restrict__ grad_prob, T *__restrict__ grad, int64_t n_tokens,
                                                                int n_expert) {
    constexpr int N = Vec<T>::N, kTokens = kBwdBlock / L;
    const int lane = threadIdx.x % L;
    const int64_t t0 = (int64_t)blockIdx.x * (kTokens * AHEAD) + threadIdx.x / L;
    Logits<T, L, V, WHOLE> a[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) a[k].load(logits, t0 + k * kTokens, n_tokens, n_expert);
    const float gl = grad_loss ? *grad_loss : 0.f, per = slope[n_expert];
    float u[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const int c = (v * L + lane) * N + i;
            const u32x4 s = load_vec<false>(slope + c, n_expert - c, false);
            const u32x4 g = grad_prob ? load_vec<false>(grad_prob + c, n_expert - c, false) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) u[v][i + j] = gl * __uint_as_float(s[j]) + __uint_as_float(g[j]) * per;
        }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
        const int64_t t = t0 + k * kTokens;
        float p[V][N], dot = 0.f;
        const float inv = a[k].softmax(p, t < n_tokens && (!mask || mask[t] == 0), n_expert);
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[v][i] *= inv;
                dot += p[v][i] * u[v][i];
            }
        dot = over_lanes<L>(dot, [](float x, float y) { return x + y; });
        if (t >= n_tokens) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * L + lane) * N;
            float out[8];
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = inv == 0.f ? 0.f : p[v][i] * (u[v][i] - dot);
            if constexpr (WHOLE) {
                if (c < n_expert) *(AnyVec *)(grad + t * n_expert + c) = Vec<T>::pack(out);
            } else {
                store_vec<false>(grad + t * n_expert + c, n_expert - c, Vec<T>::pack(out));
            }
        }
    }
}

// How a token's logits are held: f(lanes, vectors to each, whether the experts are whole vectors), integral constants
template <int N, typename F> void held_logits(int n_expert, F &&f) {
    auto is = [&](auto l, auto v) {
        if (n_expert > l.value * v.value * N) return false;
        if (n_expert % N == 0) f(l, v, std::true_type{});
        else f(l, v, std::false_type{});
        return true;
    };
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 64> wave{};
    (void)(is(one, one) || is(integral_constant<int, 2>{}, one) || is(integral_constant<int, 4>{}, one) || is(integral_constant<int, 8>{}, one) ||
           is(integral_constant<int, 16>{}, one) || is(integral_constant<int, 32>{}, one) || is(wave, one) || is(wave, integral_constant<int, 2>{}) ||
           is(wave, integral_constant<int, 4>{}) || is(wave, integral_constant<int, 8>{}) || is(wave, integral_constant<int, kMostExperts / kWave / N>{}));
}

int most_parts(int64_t n_tokens) { return (int)(n_tokens < 1 ? 1 : n_tokens < kMostParts ? n_tokens : kMostParts); }

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
    return 8 * ceil_div(n_expert, kSumCols) + 16 + (int64_t)most_parts(n_tokens) * (8 * n_expert + 8);
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
    FMOE_REQUIRE(aligned16(workspace), "%s: workspace not on 16 bytes", who);
    hipStream_t st = (hipStream_t)stream;
    const int columns = (int)ceil_div(n_expert, kSumCols), most = most_parts(n_tokens);
    Sums sums;
    sums.loss = (double *)workspace;
    sums.done = (unsigned *)(sums.loss + columns);
    sums.total = (int2 *)(sums.done + 2);
    sums.prob = (float *)(sums.total + most);
    sums.count = (int *)(sums.prob + most * n_expert);
    const Results results{expert_count, prob, slope, loss, per_slot};
    with_type(dtype, [&](auto type) {
        using T = decltype(type);
        held_logits<Vec<T>::N>((int)n_expert, [&](auto l, auto v, auto whole) {
            constexpr int kTokens = waves_of(v.value) * (kWave / l.value);
            // (what one workgroup goes through in kFewRounds rounds is not worth a second launch: 1000 x 16 float32, four rounds, 6.6 us, with
            // four workgroups and the launch that joins them 8.5; 2000 x 16, eight, 8.1 and 8.5)
            const int64_t rounds = ceil_div(n_tokens, kTokens);
            const int parts = (int)(rounds <= kFewRounds ? 1 : rounds < most ? rounds : most);
            balance_sum_kernel<T, l.value, v.value, whole.value><<<parts, waves_of(v.value) * kWave, 0, st>>>(
                (const T *)logits, topk_idx, (const uint8_t *)token_mask, sums, results, n_tokens, (int)n_expert, (int)top_k);
            if (parts > 1) balance_finish_kernel<<<columns, kSumBlock, 0, st>>>(sums, results, parts, (int)n_expert);
        });
    });
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
    bool fits = true;
    with_type(dtype, [&](auto type) {
        using T = decltype(type);
        held_logits<Vec<T>::N>((int)n_expert, [&](auto l, auto v, auto whole) {
            // (one token in flight per lane where more would leave compute units without a workgroup: 16384 x 64 float32 3.6 us, four ahead 4.5;
            // 32768 x 256 bfloat16 9.7 four ahead, one 20)
            constexpr int kTokens = kBwdBlock / l.value, kAhead = ahead_of(v.value);
            const bool ahead = n_tokens >= kBwdBlocks * kTokens * kAhead;
            const int64_t blocks = ceil_div(n_tokens, kTokens * (ahead ? kAhead : 1));
            fits = blocks <= kMostThreads / kBwdBlock;
            if (!fits) return;
            (ahead ? balance_bwd_kernel<T, l.value, v.value, whole.value, kAhead> : balance_bwd_kernel<T, l.value, v.value, whole.value, 1>)<<<
                (int)blocks, kBwdBlock, 0, (hipStream_t)stream>>>(
                (const T *)logits, (const uint8_t *)token_mask, slope, grad_loss, grad_prob, (T *)grad_logits, n_tokens, (int)n_expert);
        });
    });
    if (!fits) return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
