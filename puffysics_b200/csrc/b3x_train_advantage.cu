// b3x_train_advantage.cu -- generalised advantages and returns of a rollout
// (b3x_train.h).
#include <cmath>

#include "b3x_train_common.cuh"

using namespace b3t;

namespace {

struct Rollout {
    long long steps, envs;
    const float* rewards;
    const void *values, *terminals, *last_values;
    const int* lengths;
    float *advantages, *returns;
    long long rt, rn, vt, vn, dt, dn, ln, at, an, ot, on;
    float gamma, decay;  // gamma, gamma * lam
    int terminal_bytes;
};

__device__ __forceinline__ bool terminal(const Rollout& a, long long i) {
    return a.terminal_bytes == 4 ? ((const float*)a.terminals)[i] != 0.0f : ((const unsigned char*)a.terminals)[i] != 0;
}

// One thread an environment, from its last step to its first.
template <class V>
__global__ void __launch_bounds__(128) advantage_kernel(Rollout a) {
    const long long n = (long long)blockIdx.x * 128 + threadIdx.x;
    if (n >= a.envs) return;
    long long len = a.lengths ? a.lengths[n] : a.steps;
    len = len < 0 ? 0 : len > a.steps ? a.steps : len;
    for (long long t = a.steps - 1; t >= len; t--) {
        a.advantages[t * a.at + n * a.an] = 0.0f;
        if (a.returns) a.returns[t * a.ot + n * a.on] = 0.0f;
    }
    float after = len ? to_float(((const V*)a.last_values)[n * a.ln]) : 0.0f, ahead = 0.0f;
    for (long long t = len - 1; t >= 0; t--) {
        const float v = to_float(((const V*)a.values)[t * a.vt + n * a.vn]);
        const bool end = terminal(a, t * a.dt + n * a.dn);
        float x = a.rewards[t * a.rt + n * a.rn];
        if (!end) x += a.gamma * after;
        x -= v;
        if (!end) x += a.decay * ahead;
        ahead = x;
        after = v;
        a.advantages[t * a.at + n * a.an] = ahead;
        if (a.returns) a.returns[t * a.ot + n * a.on] = ahead + v;
    }
}

}  // namespace

int b3x_train_advantage_gpu(long long steps, long long envs, const float* rewards, const void* values, int value_type,
        const void* terminals, int terminal_type, const void* last_values, const int* lengths, float* advantages,
        float* returns, const long long strides[11], float gamma, float lam, void* stream) {
    if (steps < 0 || envs < 0 || value_type < B3X_F32 || value_type > B3X_F16 ||
        (terminal_type != B3X_F32 && terminal_type != B3X_U8) || !std::isfinite(gamma) || !std::isfinite(lam))
        return (int)cudaErrorInvalidValue;
    if (steps == 0 || envs == 0) return (int)cudaSuccess;
    const int vb = value_type == B3X_F32 ? 4 : 2, tb = terminal_type == B3X_F32 ? 4 : 1;
    if (!rewards || !values || !terminals || !last_values || !advantages || !strides || envs > 0x7fffffff ||
        steps > 0x7fffffff || (uintptr_t)rewards % 4 || (uintptr_t)values % vb || (uintptr_t)terminals % tb ||
        (uintptr_t)last_values % vb || (uintptr_t)lengths % 4 || (uintptr_t)advantages % 4 || (uintptr_t)returns % 4)
        return (int)cudaErrorInvalidValue;
    for (int i = 0; i < 11; i++)
        if (strides[i] < 0) return (int)cudaErrorInvalidValue;
    if (!apart(steps, envs, strides[7], strides[8]) || (returns && !apart(steps, envs, strides[9], strides[10])) ||
        (const void*)advantages == rewards || advantages == values || advantages == terminals || returns == advantages ||
        (returns && ((const void*)returns == rewards || returns == values || returns == terminals)))
        return (int)cudaErrorInvalidValue;
    const Rollout a{steps, envs, rewards, values, terminals, last_values, lengths, advantages, returns,
                    strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6],
                    strides[7], strides[8], strides[9], strides[10], gamma, gamma * lam, tb};
    const unsigned grid = (unsigned)((envs + 127) / 128);
    if (value_type == B3X_F32) advantage_kernel<float><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    if (value_type == B3X_BF16) advantage_kernel<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    if (value_type == B3X_F16) advantage_kernel<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    return (int)cudaGetLastError();
}
