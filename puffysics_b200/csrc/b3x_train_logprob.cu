// b3x_train_logprob.cu -- log probabilities of actions, entropies and most
// likely alternatives of rows of logits, and their gradient (b3x_train.h).
#include <cmath>

#include "b3x_train_common.cuh"

using namespace b3t;

namespace {

struct Rows {
    const void* logits;
    long long rows, row_stride;
    const unsigned char* mask;
    long long mask_stride;
    const void* actions;
    int action_bytes, width;
    float scale;
};

__device__ __forceinline__ long long action_of(const Rows& a, long long row) {
    if (!a.actions) return -1;
    return a.action_bytes == 8 ? ((const long long*)a.actions)[row] : (long long)((const int*)a.actions)[row];
}

template <class T>
__device__ __forceinline__ float logit(const Rows& a, long long row, int j) {
    if (a.mask && !a.mask[row * a.mask_stride + j]) return -kInf;
    return to_float(((const T*)a.logits)[row * a.row_stride + j]);
}

struct Out {
    float *logp, *entropy, *stats;
    int top;
    int* top_ids;
    float* top_logp;
};

constexpr int kThreads = 256;

template <class F>
__device__ float block_reduce(float x, float* buf, F f) {
    for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(~0u, x, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = x;
    __syncthreads();
    x = buf[0];
    for (int i = 1; i < kThreads / 32; i++) x = f(x, buf[i]);
    return x;
}

// One block a row: maximum, sums, then each alternative as the best one after
// the last.
template <class T>
__global__ void __launch_bounds__(kThreads) logprob_kernel(Rows a, Out o) {
    __shared__ float buf[kThreads / 32];
    __shared__ int ibuf[kThreads / 32];
    const long long row = blockIdx.x;
    float m = -kInf;
    for (int j = threadIdx.x; j < a.width; j += kThreads) m = max_nan(m, logit<T>(a, row, j));
    m = block_reduce(m, buf, [](float x, float y) { return max_nan(x, y); });
    float s = 0.0f, t = 0.0f;
    for (int j = threadIdx.x; j < a.width; j += kThreads) {
        const float d = fmaxf((logit<T>(a, row, j) - m) * a.scale, -1e4f), e = expf(d);
        s += e;
        t += e * d;
    }
    auto add = [](float x, float y) { return x + y; };
    s = block_reduce(s, buf, add);
    t = block_reduce(t, buf, add);
    const bool empty = m == -kInf;
    const float bad = empty ? 0.0f : m - m;  // NaN where the maximum is no number
    const float logsum = empty ? 0.0f : logf(s) + bad;
    if (threadIdx.x == 0) {
        if (o.stats) o.stats[2 * row] = m, o.stats[2 * row + 1] = logsum;
        if (o.entropy) o.entropy[row] = empty ? 0.0f : logsum - t / s;
        if (o.logp) {
            const long long j = action_of(a, row);
            float lp = 0.0f;
            if (j >= 0 && j < a.width) lp = empty ? -kInf : (logit<T>(a, row, (int)j) - m) * a.scale - logsum;
            o.logp[row] = lp;
        }
    }
    float last = kInf;
    int last_id = -1;
    for (int k = 0; k < o.top; k++) {
        float best = -kInf;
        int id = 0x7fffffff;
        for (int j = threadIdx.x; j < a.width; j += kThreads) {
            const float z = logit<T>(a, row, j);
            const bool after = z < last || (z == last && j > last_id);
            if (after && z > best) best = z, id = j;
        }
        const float top = block_reduce(best, buf, [](float x, float y) { return fmaxf(x, y); });
        int first = best == top ? id : 0x7fffffff;
        for (int s2 = 16; s2; s2 >>= 1) first = min(first, __shfl_xor_sync(~0u, first, s2));
        __syncthreads();
        if (threadIdx.x % 32 == 0) ibuf[threadIdx.x / 32] = first;
        __syncthreads();
        for (int i = 0; i < kThreads / 32; i++) first = min(first, ibuf[i]);
        const bool none = top == -kInf;
        last = top;
        last_id = first;
        if (threadIdx.x == 0) {
            o.top_ids[row * o.top + k] = none ? -1 : first;
            o.top_logp[row * o.top + k] = none ? -kInf : (top - m) * a.scale - logsum;
        }
    }
}

struct Grad {
    const float *stats, *entropy, *d_logp, *d_entropy;
    void* grad;
    long long grad_stride;
};

template <class T>
__global__ void __launch_bounds__(kThreads) logprob_grad_kernel(Rows a, Grad b) {
    const long long row = blockIdx.x;
    const float m = b.stats[2 * row], logsum = b.stats[2 * row + 1];
    const float h = b.d_entropy ? b.d_entropy[row] : 0.0f, H = b.d_entropy ? b.entropy[row] : 0.0f;
    const long long act = action_of(a, row);
    float g = 0.0f;
    if (b.d_logp && act >= 0 && act < a.width && logit<T>(a, row, (int)act) != -kInf) g = b.d_logp[row];
    __syncthreads();  // the action's logit may be what another thread overwrites
    T* grad = (T*)b.grad + row * b.grad_stride;
    for (int j = threadIdx.x; j < a.width; j += kThreads) {
        const float z = logit<T>(a, row, j);
        float d = 0.0f;
        if (z != -kInf) {
            const float lp = fmaxf((z - m) * a.scale - logsum, -1e4f) + (m - m), p = expf(lp);
            d = -p * (g + h * (lp + H));
            if (j == act) d += g;
        }
        grad[j] = from_float<T>(d * a.scale);
    }
}

bool rows_ok(const void* logits, int type, long long rows, long long width, long long row_stride,
             const unsigned char* mask, long long mask_stride, const void* actions, int action_bytes, float scale) {
    if (type < B3X_F32 || type > B3X_F16 || rows < 0 || rows > 0x7fffffff || !(scale > 0.0f) || !std::isfinite(scale))
        return false;
    if (rows == 0) return true;
    if (width < 1 || width > (1ll << 30) || row_stride < 0 || mask_stride < 0 || !logits) return false;
    if ((uintptr_t)logits % (type == B3X_F32 ? 4 : 2)) return false;
    if (actions && action_bytes != 4 && action_bytes != 8) return false;
    return !actions || (uintptr_t)actions % action_bytes == 0;
}

bool aligned4(const void* p) { return (uintptr_t)p % 4 == 0; }

}  // namespace

int b3x_train_logprob_gpu(const void* logits, int type, long long rows, long long width, long long row_stride,
        const unsigned char* mask, long long mask_stride, const void* actions, int action_bytes, float scale,
        float* logp, float* entropy, float* stats, int top, int* top_ids, float* top_logp, void* stream) {
    if (!rows_ok(logits, type, rows, width, row_stride, mask, mask_stride, actions, action_bytes, scale) || top < 0 ||
        top > B3X_TRAIN_MAX_TOP)
        return (int)cudaErrorInvalidValue;
    if (rows == 0) return (int)cudaSuccess;
    if ((logp && !actions) || (top && (!top_ids || !top_logp)) || (!logp && !entropy && !stats && !top) ||
        !aligned4(logp) || !aligned4(entropy) || !aligned4(stats) || !aligned4(top_ids) || !aligned4(top_logp))
        return (int)cudaErrorInvalidValue;
    const Rows a{logits, rows, row_stride, mask, mask_stride, actions, action_bytes, (int)width, scale};
    const Out o{logp, entropy, stats, top, top_ids, top_logp};
    const unsigned grid = (unsigned)rows;
    if (type == B3X_F32) logprob_kernel<float><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, o);
    if (type == B3X_BF16) logprob_kernel<__nv_bfloat16><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, o);
    if (type == B3X_F16) logprob_kernel<__half><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, o);
    return (int)cudaGetLastError();
}

int b3x_train_logprob_grad_gpu(const void* logits, int type, long long rows, long long width, long long row_stride,
        const unsigned char* mask, long long mask_stride, const void* actions, int action_bytes, float scale,
        const float* stats, const float* entropy, const float* d_logp, const float* d_entropy, void* grad,
        long long grad_stride, void* stream) {
    if (!rows_ok(logits, type, rows, width, row_stride, mask, mask_stride, actions, action_bytes, scale))
        return (int)cudaErrorInvalidValue;
    if (rows == 0) return (int)cudaSuccess;
    if (!stats || !grad || (d_logp && !actions) || (d_entropy && !entropy) || !aligned4(stats) || !aligned4(entropy) ||
        !aligned4(d_logp) || !aligned4(d_entropy) || (uintptr_t)grad % (type == B3X_F32 ? 4 : 2) ||
        !apart(rows, width, grad_stride, 1) || (grad == logits && rows > 1 && grad_stride != row_stride))
        return (int)cudaErrorInvalidValue;
    const Rows a{logits, rows, row_stride, mask, mask_stride, actions, action_bytes, (int)width, scale};
    const Grad b{stats, entropy, d_logp, d_entropy, grad, grad_stride};
    const unsigned grid = (unsigned)rows;
    if (type == B3X_F32) logprob_grad_kernel<float><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, b);
    if (type == B3X_BF16) logprob_grad_kernel<__nv_bfloat16><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, b);
    if (type == B3X_F16) logprob_grad_kernel<__half><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a, b);
    return (int)cudaGetLastError();
}
