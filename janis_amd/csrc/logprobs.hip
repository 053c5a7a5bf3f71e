// Log probabilities of rows of logits: given tokens, the entropy, the likeliest tokens.
#include "jh_common.hpp"

namespace jh {
namespace {

__device__ __forceinline__ float logit(const LogProbsArgs& a, int64_t row, int i) {
    const int64_t at = row * a.stride + i;
    return a.f32 ? static_cast<const float*>(a.x)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.x)[at]);
}

// Order of a value and its token as one number: larger values first, of equal ones the
// lower token; 0 is below all of them (NaN and -inf).
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    if (!(v > -__builtin_inff())) return 0;
    const uint32_t u = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return (uint64_t)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// A block to a row; its maximum, its sums, then its tokens one after the other.
constexpr int kThreads = 1024;
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogProbsArgs a) {
    __shared__ float s_f[3][16];
    __shared__ uint64_t s_k[16];
    __shared__ int s_ids[JH_LOGPROBS_TOP];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -__builtin_inff(), bad = 0.0f;
    for (int i = tid; i < a.vocab; i += kThreads) {
        const float x = logit(a, row, i);
        m = fmaxf(m, x);
        bad += x != x ? 1.0f : 0.0f;
    }
    m = wave_max(m), bad = wave_sum(bad);
    if (lane == 0) s_f[0][wave] = m, s_f[1][wave] = bad;
    __syncthreads();
    for (int w = 0; w < 16; w++) m = fmaxf(m, s_f[0][w]), bad += w == wave ? 0.0f : s_f[1][w];
    __syncthreads();
    float sum = 0.0f, sumd = 0.0f;
    for (int i = tid; i < a.vocab; i += kThreads) {
        const float d = (logit(a, row, i) - m) * a.scale, e = expf(d);
        sum += e;
        if (e > 0.0f) sumd += e * d;
    }
    sum = wave_sum(sum), sumd = wave_sum(sumd);
    if (lane == 0) s_f[0][wave] = sum, s_f[1][wave] = sumd;
    __syncthreads();
    sum = sumd = 0.0f;
    for (int w = 0; w < 16; w++) sum += s_f[0][w], sumd += s_f[1][w];
    const bool none = bad > 0.0f || !(m > -__builtin_inff()) || !(m < __builtin_inff());
    const float ln = none ? __builtin_nanf("") : logf(sum);
    if (tid < a.n_tokens) {
        const int t = a.tokens[row * a.n_tokens + tid];
        const bool is = t >= 0 && t < a.vocab;
        a.logprobs[row * a.n_tokens + tid] = is ? (logit(a, row, t) - m) * a.scale - ln : __builtin_nanf("");
    }
    if (tid == 0 && a.entropy) a.entropy[row] = ln - sumd / sum;
    uint64_t last = ~0ull;
    int n = 0;  // tokens found (the rest: the lowest that are not among them)
    for (int j = 0; j < a.top_k; j++) {
        uint64_t best = 0;
        if (last)
            for (int i = tid; i < a.vocab; i += kThreads) {
                const uint64_t k = key_of(logit(a, row, i), i);
                if (k < last && k > best) best = k;
            }
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t other = (uint64_t)(uint32_t)__shfl_xor((int)(best >> 32), d, 64) << 32 | (uint32_t)__shfl_xor((int)best, d, 64);
            best = best > other ? best : other;
        }
        __syncthreads();
        if (lane == 0) s_k[wave] = best;
        __syncthreads();
        for (int w = 0; w < 16; w++) best = best > s_k[w] ? best : s_k[w];
        last = best;
        if (best) n = j + 1;
        if (tid == 0) {
            float v = -__builtin_inff();
            int id = (int)~(uint32_t)best;
            if (best) {
                v = value_of(best);
            } else {
                id = j == n ? -1 : s_ids[j - 1];
                bool taken = true;
                while (taken) {
                    id++;
                    taken = false;
                    for (int i = 0; i < n; i++) taken |= s_ids[i] == id;
                }
            }
            s_ids[j] = id;
            a.top_ids[row * a.top_k + j] = id;
            a.top_logprobs[row * a.top_k + j] = (v - m) * a.scale - ln;
        }
    }
}

}  // namespace

size_t logprobs_workspace_bytes(const LogProbsArgs&, int) { return 0; }

Status launch_logprobs(const LogProbsArgs& a, void*, int, hipStream_t st) {
    hipLaunchKernelGGL(logprobs_kernel, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a);
    return Status::ok();
}

}  // namespace jh
