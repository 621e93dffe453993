// b3x_train_logprob_grad.cu -- the gradient of action log probabilities and
// entropies with respect to rows of logits (b3x_train.h).
#include "b3x_train_rows.cuh"

using namespace b3t;

namespace {

struct Grad {
    const float *stats, *entropy, *d_logp, *d_entropy;
    void* grad;
    long long grad_stride;
};

__device__ __forceinline__ uint32_t pack_pair(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&a);
}
__device__ __forceinline__ uint32_t pack_pair(float x, float y, __half) {
    const __half2 a = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&a);
}

constexpr int kThreads = 512;
constexpr int kUnroll = 4;
constexpr int kMaxCluster = 8;

// 2^bits threads a row (a cluster's blocks together where it has more than one),
// 16 bytes of logits and of gradients at a time; bound by memory (2,048 rows of
// 65,536 bf16: 92 us, 5.8 TB/s, 90% of the copy rate; 4,096 rows of 50,001: 157
// us, 81%; 2,048 masked rows of 50,001 f16 131 us, 60%: every vector's mask is
// two or three loads of a word and their shifts).  Gradients at another place
// modulo 16 bytes than their logits are stored one by one (500 us for the 157 of
// 4,096 rows of 50,001).  With
// e = log p_j the gradient is p_j (B e + A) with A = -scale (g + h H) and
// B = -scale h, and scale g more at the action.
template <class T, bool kMask>
__global__ void __launch_bounds__(kThreads, 2) grad_kernel(const Rows a, const Grad b, const int bits, const int cluster) {
    constexpr int N = Vec<T>::n;
    int part = 0;
    if (cluster > 1) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    const int lane = (threadIdx.x & ((1 << bits) - 1)) + part * blockDim.x, lanes = (1 << bits) * cluster;
    const long long row = (long long)(blockIdx.x / cluster) * (blockDim.x >> bits) + (threadIdx.x >> bits);
    const bool on = row < a.rows;
    const Source<T, kMask> src(a, on ? row : 0);
    const int nv = on ? src.vectors() : 0;
    float m = 0.0f, logsum = 0.0f, g = 0.0f, h = 0.0f, H = 0.0f;
    long long act = -1;
    if (on) {
        m = b.stats[2 * row], logsum = b.stats[2 * row + 1];
        if (b.d_entropy) h = b.d_entropy[row], H = b.entropy[row];
        act = action_of(a, row);
        if (b.d_logp && act >= 0 && act < a.width) {
            if (logit<T>(a, row, (int)act) != -kInf) g = b.d_logp[row];
            else act = -1;
        } else {
            act = -1;
        }
    }
    // the action's logit is read by all before one of them overwrites it
    if (cluster > 1) asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
    else if (bits > 5) __syncthreads();
    else __syncwarp();
    T* const grad = (T*)b.grad + (on ? row : 0) * b.grad_stride;
    const bool even = (int)((uintptr_t)grad % 16 / sizeof(T)) == src.head;
    const bool sums = m - m == 0.0f;                  // else nothing is allowed, or the row is NaN
    const int at = act < 0 ? -1 : (int)act + src.head;   // the action's place among the vectors' elements
    const uint64_t minus = pack2(-m, -m), scale = pack2(a.scale, a.scale), less = pack2(-logsum, -logsum),
                   log2e = pack2(kLog2e, kLog2e);
    const float fa = -a.scale * __fmaf_rn(h, H, g), fb = -a.scale * h;
    const uint64_t A = pack2(fa, fa), B = pack2(fb, fb);
    for (int base = 0; base < nv; base += lanes * kUnroll) {
        uint4 q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int v = base + u * lanes + lane;
            if (v >= 2 && v < src.last()) q[u] = src.inner(v);
            else if (v < nv) q[u] = src.load(v);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int v = base + u * lanes + lane;
            if (v >= nv) continue;
            float d[N];
            if (sums) {
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const uint64_t z = pack2(element<T>(q[u], i), element<T>(q[u], i + 1));
                    const uint64_t e = fma2(add2(z, minus), scale, less);
                    const float2 x = unpack2(mul2(e, log2e)), f = unpack2(e);
                    const float2 y = unpack2(mul2(pack2(exp2_fast(x.x), exp2_fast(x.y)), fma2(B, e, A)));
                    d[i] = f.x > -200.0f ? y.x : 0.0f;   // p is 0 there, and e may be -infinity
                    d[i + 1] = f.y > -200.0f ? y.y : 0.0f;
                }
                if (at / N == v && at >= 0) {
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (at % N == i) d[i] = __fmaf_rn(a.scale, g, d[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) d[i] = element<T>(q[u], i) == -kInf ? 0.0f : m - m;
            }
            const int j = v * N - src.head;
            if (even && j >= 0 && j + N <= src.width) {
                uint4 w;
                if constexpr (sizeof(T) == 4) w = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
                else w = make_uint4(pack_pair(d[0], d[1], T()), pack_pair(d[2 % N], d[3 % N], T()), pack_pair(d[4 % N], d[5 % N], T()), pack_pair(d[6 % N], d[7 % N], T()));
                __stcs(reinterpret_cast<uint4*>(grad + j), w);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (j + i >= 0 && j + i < src.width) grad[j + i] = from_float<T>(d[i]);
            }
        }
    }
}

// Up to 8 logits: one thread a row (262,144 rows of 3 f32: 4.0 us, the bytes alone 2.1).
constexpr int kShort = 8;
constexpr int kShortThreads = 128;

template <class T>
__global__ void __launch_bounds__(kShortThreads) grad_short_kernel(const Rows a, const Grad b) {
    const long long row = (long long)blockIdx.x * kShortThreads + threadIdx.x;
    if (row >= a.rows) return;
    float z[kShort];
#pragma unroll
    for (int i = 0; i < kShort; i++) z[i] = i < a.width ? logit<T>(a, row, i) : -kInf;
    const float m = b.stats[2 * row], logsum = b.stats[2 * row + 1];
    const float h = b.d_entropy ? b.d_entropy[row] : 0.0f, H = b.d_entropy ? b.entropy[row] : 0.0f;
    const long long act = action_of(a, row);
    float g = 0.0f;
    if (b.d_logp) {
#pragma unroll
        for (int i = 0; i < kShort; i++)
            if (act == i && z[i] != -kInf) g = b.d_logp[row];
    }
    const float A = -a.scale * __fmaf_rn(h, H, g), B = -a.scale * h;
    T* const grad = (T*)b.grad + row * b.grad_stride;
#pragma unroll
    for (int i = 0; i < kShort; i++) {
        if (i >= a.width) break;
        const float e = __fmaf_rn(z[i] - m, a.scale, -logsum);
        float d = e > -200.0f ? exp2_fast(e * kLog2e) * __fmaf_rn(B, e, A) : 0.0f;
        if (act == i && g != 0.0f) d = __fmaf_rn(a.scale, g, d);
        if (!(m - m == 0.0f)) d = z[i] == -kInf ? 0.0f : m - m;
        grad[i] = from_float<T>(d);
    }
}

template <class T, bool kMask>
int launch_grad(const Rows& a, const Grad& b, cudaStream_t s) {
    const int nv = (int)(((long long)a.width + Vec<T>::n - 1) / Vec<T>::n) + 1;
    // Threads for a row, eight vectors each where there are enough for all SMs (65,536 rows of 1,000 bf16 56 us; with
    // four vectors 61, with two 86, with one 131), else two, and no more than a block; a cluster where rows leave SMs
    // idle (8 rows of 131,072: 4.0 us, by single blocks 12.9).
    const int each = a.rows * nv >= 148ll * 1024 * 8 ? 8 : 2;
    int bits = 0;
    while ((1 << bits) < kThreads && each << bits < nv) bits++;
    int cluster = 1;
    while (bits == 9 && cluster < kMaxCluster && a.rows * cluster * 2 <= 296 && nv >= kThreads * cluster * 2) cluster *= 2;
    const int threads = bits > 8 ? kThreads : 256;
    const long long blocks = (a.rows * (1ll << bits) + threads - 1) / threads * cluster;
    if (blocks > 0x7fffffff) return (int)cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, grad_kernel<T, kMask>, a, b, bits, cluster);
}

template <class T>
int launch(const Rows& a, const Grad& b, cudaStream_t s) {
    if (a.width <= kShort) {
        grad_short_kernel<T><<<(unsigned)((a.rows + kShortThreads - 1) / kShortThreads), kShortThreads, 0, s>>>(a, b);
        return (int)cudaGetLastError();
    }
    return a.mask ? launch_grad<T, true>(a, b, s) : launch_grad<T, false>(a, b, s);
}

}  // namespace

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
    if (type == B3X_F32) return launch<float>(a, b, (cudaStream_t)stream);
    if (type == B3X_BF16) return launch<__nv_bfloat16>(a, b, (cudaStream_t)stream);
    return launch<__half>(a, b, (cudaStream_t)stream);
}
