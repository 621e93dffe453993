// b3x_train_adamw.cu -- the global norm of a list of gradients and one AdamW
// step over a list of tensors (b3x_train.h).
#include <cmath>

#include "b3x_train_common.cuh"

using namespace b3t;

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = kThreads * 8;    // elements a block takes at a time; a multiple of B3X_TRAIN_BLOCK
constexpr int kList = 256;              // tensors of one launch: the table travels in the kernel's parameters
constexpr int kNormBlocks = 592;        // partial sums of the norm
static_assert(kChunk % B3X_TRAIN_BLOCK == 0, "a scale's elements stay in one block");

struct Tensor {
    void* p;
    const void* g;
    void *m, *v;
    float* scales;
    __nv_bfloat16* copy;
    long long n;
    float keep;          // 1 - lr weight_decay
    unsigned key;        // the tensor's part of the rounding hash
};

template <int N>
struct List {
    int count;
    unsigned first[N + 1];   // first chunk of each tensor
    Tensor t[N];
};

struct Hyper {
    float b1, c1, b2, c2, rate, root, eps;
    const float* grad_scale;
};

// The tensor that `chunk` belongs to.
template <int N>
__device__ __forceinline__ int find(const List<N>& list, unsigned chunk) {
    int lo = 0, hi = list.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

__host__ __device__ __forceinline__ unsigned mix(unsigned x) {
    x ^= x >> 16;
    x *= 0x85A308D3u;
    x ^= x >> 13;
    x *= 0x243F6A89u;
    return x ^ (x >> 16);
}

// e4m3 codes of x / scale.  Scaled by 2^-120 the format's exponents are
// float's, subnormals included, so the code is the upper bits of the word; what
// is added to the 20 bits below it rounds.
__device__ __forceinline__ unsigned encode(float y, bool stochastic, unsigned bits16) {
    unsigned w = __float_as_uint(fabsf(y) * 0x1p-120f);
    w += stochastic ? (bits16 << 4 | 8u) : 0x7FFFFu + ((w >> 20) & 1u);
    w = min(w >> 20, 0x7Eu);
    return y < 0.0f ? w | 0x80u : w;
}

__device__ __forceinline__ float decode(unsigned code) {
    const float y = __uint_as_float((code & 0x7Fu) << 20) * 0x1p120f;
    return code & 0x80u ? -y : y;
}

__device__ __forceinline__ float warp_most(float x) {
    for (int o = 16; o; o >>= 1) x = max_nan(x, __shfl_xor_sync(~0u, x, o));
    return x;
}

// A warp takes the elements of one scale at a time, eight apart by 32 for each
// lane; every operation rounds by itself (the plain formula's bits).
template <class P, class G, bool kF8, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ List<N> list, const Hyper h,
                                                         const int stochastic) {
    const float gs = h.grad_scale ? *h.grad_scale : 1.0f;
    if (!(fabsf(gs) < kInf)) return;
    const Tensor& t = list.t[find(list, blockIdx.x)];
    const unsigned chunk = blockIdx.x - list.first[&t - list.t];
    const int lane = threadIdx.x % 32;
    const long long base = (long long)chunk * kChunk + threadIdx.x / 32 * B3X_TRAIN_BLOCK;
    if (base >= t.n) return;
    float m[8], r[8];
    float sm = 1.0f, sr = 1.0f;
    if (kF8) sm = t.scales[base / B3X_TRAIN_BLOCK * 2], sr = t.scales[base / B3X_TRAIN_BLOCK * 2 + 1];
    float most_m = 0.0f, most_r = 0.0f;
    for (int k = 0; k < 8; k++) {
        const long long i = base + k * 32 + lane;
        m[k] = r[k] = 0.0f;
        if (i >= t.n) continue;
        const float g = to_float(((const G*)t.g)[i]) * gs;
        float v;
        if (kF8) {
            m[k] = decode(((unsigned char*)t.m)[i]) * sm;
            v = decode(((unsigned char*)t.v)[i]) * sr;
            v = v * v;
        } else {
            m[k] = ((float*)t.m)[i];
            v = ((float*)t.v)[i];
        }
        m[k] = m[k] * h.b1 + g * h.c1;
        v = v * h.b2 + (g * g) * h.c2;
        r[k] = sqrtf(v);
        if (!kF8) ((float*)t.m)[i] = m[k], ((float*)t.v)[i] = v;
        float p = to_float(((P*)t.p)[i]) * t.keep - (m[k] / (r[k] * h.root + h.eps)) * h.rate;
        if (t.copy) t.copy[i] = __float2bfloat16_rn(p);
        if (sizeof(P) == 2 && stochastic && fabsf(p) < kInf) {
            const unsigned low = mix(mix((unsigned)i * 0x9E3779B1u + (unsigned)(i >> 32) * 0x6A09E667u + t.key) + 0x9E3779B1u);
            p = __uint_as_float((__float_as_uint(p) + (low & 0xFFFFu)) & 0xFFFF0000u);
        }
        ((P*)t.p)[i] = from_float<P>(p);
        most_m = max_nan(most_m, fabsf(m[k]));
        most_r = max_nan(most_r, r[k]);
    }
    if (!kF8) return;
    most_m = warp_most(most_m), most_r = warp_most(most_r);
    const bool zm = most_m < 0x1p-100f, zr = most_r < 0x1p-100f;   // false for NaN
    const float im = zm ? 0.0f : 448.0f / most_m, ir = zr ? 0.0f : 448.0f / most_r;
    if (lane == 0) {
        t.scales[base / B3X_TRAIN_BLOCK * 2] = zm ? 0.0f : most_m / 448.0f;
        t.scales[base / B3X_TRAIN_BLOCK * 2 + 1] = zr ? 0.0f : most_r / 448.0f;
    }
    for (int k = 0; k < 8; k++) {
        const long long i = base + k * 32 + lane;
        if (i >= t.n) break;
        const unsigned bits = mix((unsigned)i * 0x9E3779B1u + (unsigned)(i >> 32) * 0x6A09E667u + t.key);
        ((unsigned char*)t.m)[i] = (unsigned char)encode(m[k] * im, stochastic, bits & 0xFFFFu);
        unsigned c = encode(r[k] * ir, stochastic, bits >> 16);
        if (c == 0 && r[k] > 0.0f && !zr) c = 1;
        ((unsigned char*)t.v)[i] = (unsigned char)c;
    }
}

// Each block's chunks, then the blocks' sums by one block, in 64 bits.
template <class G, int N>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ List<N> list, double* sums, int more) {
    __shared__ double buf[kThreads / 32];
    double s = 0.0;
    const unsigned chunks = list.first[list.count];
    for (unsigned c = blockIdx.x; c < chunks; c += kNormBlocks) {
        const int k = find(list, c);
        const Tensor& t = list.t[k];
        const long long base = (long long)(c - list.first[k]) * kChunk;
        for (int u = 0; u < 8; u++) {
            const long long i = base + u * kThreads + threadIdx.x;
            if (i < t.n) {
                const double g = (double)to_float(((const G*)t.g)[i]);
                s += g * g;
            }
        }
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / 32; i++) s += buf[i];
        sums[blockIdx.x] = more ? sums[blockIdx.x] + s : s;
    }
}

__global__ void __launch_bounds__(32) norm_end_kernel(const double* sums, float max_norm, float* out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < kNormBlocks; i += 32) s += sums[i];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(s);
        out[0] = norm;
        out[1] = fabsf(norm) < kInf ? fminf(1.0f, max_norm / (norm + 1e-6f)) : norm - norm;
    }
}

int bytes_of(int type) { return type == B3X_F32 ? 4 : type == B3X_E4M3 || type == B3X_U8 ? 1 : 2; }

bool at(const void* p, int bytes) { return p && (uintptr_t)p % bytes == 0; }

// Fills lists of at most N tensors and hands each to `go`; tensors without elements are left out.
template <int N, class Fill, class Go>
int each_list(int count, const long long* sizes, Fill fill, Go go) {
    static thread_local List<N> list;
    int k = 0;
    bool more = false;
    while (k < count) {
        list.count = 0;
        list.first[0] = 0;
        for (; k < count && list.count < N; k++) {
            if (sizes[k] == 0) continue;
            const long long chunks = (sizes[k] + kChunk - 1) / kChunk;
            if (list.first[list.count] + chunks > 0x7fffffff) break;
            list.t[list.count] = fill(k);
            list.first[list.count + 1] = list.first[list.count] + (unsigned)chunks;
            list.count++;
        }
        if (list.count == 0) break;
        go(list, more);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int)e;
        more = true;
    }
    return (int)cudaSuccess;
}

bool sizes_ok(int count, const long long* sizes) {
    if (count < 0 || (count > 0 && !sizes)) return false;
    for (int k = 0; k < count; k++)
        if (sizes[k] < 0 || sizes[k] > (1ll << 40)) return false;
    return true;
}

}  // namespace

size_t b3x_train_grad_norm_workspace_bytes(void) { return kNormBlocks * sizeof(double); }

int b3x_train_grad_norm_gpu(int count, const void* const* grads, int grad_type, const long long* sizes,
        double max_norm, float* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!sizes_ok(count, sizes) || grad_type < B3X_F32 || grad_type > B3X_F16 || !(max_norm > 0.0) || !at(out, 4) ||
        !at(workspace, 8) || workspace_bytes < b3x_train_grad_norm_workspace_bytes() || (count > 0 && !grads))
        return (int)cudaErrorInvalidValue;
    for (int k = 0; k < count; k++)
        if (sizes[k] > 0 && !at(grads[k], bytes_of(grad_type))) return (int)cudaErrorInvalidValue;
    double* sums = (double*)workspace;
    const cudaStream_t s = (cudaStream_t)stream;
    bool any = false;
    const int e = each_list<kList>(
        count, sizes,
        [&](int k) { return Tensor{nullptr, grads[k], nullptr, nullptr, nullptr, nullptr, sizes[k], 0.0f, 0}; },
        [&](const List<kList>& list, bool more) {
            any = true;
            if (grad_type == B3X_F32) norm_kernel<float><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
            if (grad_type == B3X_BF16) norm_kernel<__nv_bfloat16><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
            if (grad_type == B3X_F16) norm_kernel<__half><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
        });
    if (e) return e;
    if (!any) {
        const cudaError_t z = cudaMemsetAsync(sums, 0, kNormBlocks * sizeof(double), s);
        if (z != cudaSuccess) return (int)z;
    }
    norm_end_kernel<<<1, 32, 0, s>>>(sums, (float)max_norm, out);
    return (int)cudaGetLastError();
}

int b3x_train_adamw_gpu(int count, void* const* params, int param_type, const void* const* grads, int grad_type,
        void* const* exp_avg, void* const* exp_avg_sq, float* const* scales, int state_type, void* const* copies,
        const long long* sizes, const float* decays, long long step, double lr, double beta1, double beta2, double eps,
        double weight_decay, const float* grad_scale, int stochastic, unsigned seed, void* stream) {
    const bool f8 = state_type == B3X_E4M3;
    if (!sizes_ok(count, sizes) || (param_type != B3X_F32 && param_type != B3X_BF16) || grad_type < B3X_F32 ||
        grad_type > B3X_F16 || (state_type != B3X_F32 && !f8) || step < 1 || !std::isfinite(lr) || !(beta1 >= 0.0) ||
        !(beta1 < 1.0) || !(beta2 >= 0.0) || !(beta2 < 1.0) || !(eps >= 0.0) || !std::isfinite(eps) ||
        !std::isfinite(weight_decay) || (grad_scale && !at(grad_scale, 4)))
        return (int)cudaErrorInvalidValue;
    if (count == 0) return (int)cudaSuccess;
    if (!params || !grads || !exp_avg || !exp_avg_sq || (f8 && !scales)) return (int)cudaErrorInvalidValue;
    for (int k = 0; k < count; k++) {
        if (decays && !std::isfinite(decays[k])) return (int)cudaErrorInvalidValue;
        if (sizes[k] == 0) continue;
        const int sb = bytes_of(state_type);
        if (!at(params[k], bytes_of(param_type)) || !at(grads[k], bytes_of(grad_type)) || !at(exp_avg[k], sb) ||
            !at(exp_avg_sq[k], sb) || (f8 && !at(scales[k], 8)) ||
            (copies && copies[k] && !at(copies[k], 2)))
            return (int)cudaErrorInvalidValue;
    }
    const double t = (double)step;
    const Hyper h{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2),
                  (float)(lr / (1.0 - std::pow(beta1, t))), (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, t))),
                  (float)eps, grad_scale};
    const cudaStream_t s = (cudaStream_t)stream;
    auto fill = [&](int k) {
        const double wd = decays ? (double)decays[k] : weight_decay;
        const unsigned key = mix(seed + (unsigned)k * 0x9E3779B1u + (unsigned)(unsigned long long)step * 0x6A09E667u);
        return Tensor{params[k], grads[k], exp_avg[k], exp_avg_sq[k], f8 ? scales[k] : nullptr,
                      copies ? (__nv_bfloat16*)copies[k] : nullptr, sizes[k], (float)(1.0 - lr * wd), key};
    };
    auto go = [&](const auto& list, bool) {
        const unsigned grid = list.first[list.count];
#define B3T_GO(P, G) \
        (f8 ? adamw_kernel<P, G, true><<<grid, kThreads, 0, s>>>(list, h, stochastic) \
            : adamw_kernel<P, G, false><<<grid, kThreads, 0, s>>>(list, h, stochastic))
        if (param_type == B3X_F32) {
            if (grad_type == B3X_F32) B3T_GO(float, float);
            if (grad_type == B3X_BF16) B3T_GO(float, __nv_bfloat16);
            if (grad_type == B3X_F16) B3T_GO(float, __half);
        } else {
            if (grad_type == B3X_F32) B3T_GO(__nv_bfloat16, float);
            if (grad_type == B3X_BF16) B3T_GO(__nv_bfloat16, __nv_bfloat16);
            if (grad_type == B3X_F16) B3T_GO(__nv_bfloat16, __half);
        }
#undef B3T_GO
    };
    return each_list<kList>(count, sizes, fill, go);
}
