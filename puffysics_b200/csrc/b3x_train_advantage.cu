// b3x_train_advantage.cu -- generalised advantages and returns of a rollout
// (b3x_train.h).
//
// A_t = x_t + a_t A_{t+1} with x_t = delta_t and a_t = gamma lam, or nothing
// after x_t where the step ends an episode or is an environment's last: a_t is
// NaN there, which any product with it stays.  Steps in a row compose to
// a pair (a, b) too, A = b + a A_after, and pairs compose associatively; so time
// is split over threads: each composes a few consecutive steps in registers, a
// suffix scan over lanes, warps and blocks gives each thread the A after its
// steps, and it walks back through them.  Inputs are read once and outputs
// written once; bound by memory for large rollouts and by the launch and one
// trip to memory for those of an environment batch.  Where a is NaN nothing is
// multiplied: what lies beyond a terminal may be NaN itself.  A product of many
// gamma lam never becomes 0: a NaN or infinity reaches every step before it,
// back to a terminal, however the steps are split.
#include <cmath>

#include "b3x_train_common.cuh"

using namespace b3t;

namespace {

struct Rollout {
    int steps, envs;
    const float* rewards;
    const void *values, *terminals, *last_values;
    const int* lengths;
    float *advantages, *returns;
    long long rt, rn, vt, vn, dt, dn, ln, at, an, ot, on;
    float gamma, decay;  // gamma, gamma * lam (kCut where that is 0)
};

constexpr float kCut = __builtin_nanf("");

// A = b + a A_after, or b where a is NaN.
struct Pair {
    float a, b;
};
__device__ __forceinline__ float apply(Pair p, float after) { return p.a == p.a ? __fmaf_rn(p.a, after, p.b) : p.b; }
// A product that fell to 0 becomes the least of the floats.
__device__ __forceinline__ float not_zero(float a) {
    float y;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(0x1p-149f));
    return y;
}
__device__ __forceinline__ Pair compose(Pair first, Pair then) { return Pair{not_zero(first.a * then.a), apply(first, then.b)}; }

// kSteps consecutive steps of one environment, from t on.  A step outside the
// rollout leaves A as it is (a = 1, x = 0); one beyond its environment's end has
// A = 0 (a = kCut, x = 0).
template <int kSteps>
struct Steps {
    float x[kSteps], a[kSteps], v[kSteps];

    __device__ __forceinline__ Pair pair() const {
        Pair p{a[kSteps - 1], x[kSteps - 1]};
#pragma unroll
        for (int i = kSteps - 2; i >= 0; i--) p = Pair{a[i] * p.a, apply(Pair{a[i], x[i]}, p.b)};
        p.a = not_zero(p.a);
        return p;
    }
};

template <class V> __device__ __forceinline__ float4 load4(const V* p);
template <> __device__ __forceinline__ float4 load4(const float* p) { return __ldcs(reinterpret_cast<const float4*>(p)); }
template <> __device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float4 load4(const __half* p) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <> __device__ __forceinline__ float4 load4(const unsigned char* p) {
    const unsigned w = __ldcs(reinterpret_cast<const unsigned*>(p));
    return make_float4((float)(w & 0xFF), (float)(w >> 8 & 0xFF), (float)(w >> 16 & 0xFF), (float)(w >> 24));
}

// Steps [t, t + kSteps) of environment n, of which len count.  kVec: time is
// consecutive in memory and t is on a 4-element boundary of every array.
template <class V, class D, int kSteps, bool kVec>
__device__ __forceinline__ Steps<kSteps> load_steps(const Rollout& a, int n, int t, int len) {
    Steps<kSteps> s;
    const float* r = a.rewards + (long long)n * a.rn + (long long)t * a.rt;
    const V* v = (const V*)a.values + (long long)n * a.vn + (long long)t * a.vt;
    const D* d = (const D*)a.terminals + (long long)n * a.dn + (long long)t * a.dt;
    bool end[kSteps];
    const bool whole = t >= 0 && t + kSteps <= len;
    if (whole) {
        const float after = t + kSteps < len ? to_float(v[(long long)kSteps * a.vt]) : to_float(((const V*)a.last_values)[n * a.ln]);
        if (kVec) {
#pragma unroll
            for (int i = 0; i < kSteps; i += 4) {
                const float4 x = load4(r + i), y = load4(v + i), z = load4(d + i);
                s.x[i] = x.x, s.x[i + 1] = x.y, s.x[i + 2] = x.z, s.x[i + 3] = x.w;
                s.v[i] = y.x, s.v[i + 1] = y.y, s.v[i + 2] = y.z, s.v[i + 3] = y.w;
                end[i] = z.x != 0.0f, end[i + 1] = z.y != 0.0f, end[i + 2] = z.z != 0.0f, end[i + 3] = z.w != 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                s.x[i] = __ldcs(r), s.v[i] = to_float(*v), end[i] = *d != (D)0;
                r += a.rt, v += a.vt, d += a.dt;
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
            const float next = i == kSteps - 1 ? after : s.v[i + 1];
            s.x[i] = (end[i] ? s.x[i] : __fmaf_rn(a.gamma, next, s.x[i])) - s.v[i];
            s.a[i] = end[i] ? kCut : a.decay;
        }
        if (t + kSteps == len) s.a[kSteps - 1] = kCut;
        return s;
    }
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int k = t + i;
        s.x[i] = s.v[i] = 0.0f;
        s.a[i] = k >= 0 && k < a.steps ? kCut : 1.0f;
        if (k >= 0 && k < len) {
            const float next = k + 1 < len ? to_float(v[(long long)(i + 1) * a.vt]) : to_float(((const V*)a.last_values)[n * a.ln]);
            const bool over = d[(long long)i * a.dt] != (D)0;
            s.v[i] = to_float(v[(long long)i * a.vt]);
            s.x[i] = r[(long long)i * a.rt];
            s.x[i] = (over ? s.x[i] : __fmaf_rn(a.gamma, next, s.x[i])) - s.v[i];
            s.a[i] = over || k + 1 == len ? kCut : a.decay;
        }
    }
    return s;
}

template <int kSteps, bool kVec>
__device__ __forceinline__ void store_steps(const Rollout& a, const Steps<kSteps>& s, int n, int t, int len, float after) {
    float A[kSteps];
#pragma unroll
    for (int i = kSteps - 1; i >= 0; i--) A[i] = after = apply(Pair{s.a[i], s.x[i]}, after);
    float* adv = a.advantages + (long long)n * a.an + (long long)t * a.at;
    float* ret = a.returns ? a.returns + (long long)n * a.on + (long long)t * a.ot : nullptr;
    // beyond the environment's end A, x and v are 0 already
    if (t >= 0 && t + kSteps <= a.steps && (t + kSteps <= len || t >= len)) {
        if (kVec) {
#pragma unroll
            for (int i = 0; i < kSteps; i += 4) {
                __stcs(reinterpret_cast<float4*>(adv + i), make_float4(A[i], A[i + 1], A[i + 2], A[i + 3]));
                if (ret)
                    __stcs(reinterpret_cast<float4*>(ret + i),
                           make_float4(A[i] + s.v[i], A[i + 1] + s.v[i + 1], A[i + 2] + s.v[i + 2], A[i + 3] + s.v[i + 3]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                __stcs(adv, A[i]);
                adv += a.at;
                if (ret) {
                    __stcs(ret, A[i] + s.v[i]);
                    ret += a.ot;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        if (t + i < 0 || t + i >= a.steps) continue;
        adv[(long long)i * a.at] = A[i];
        if (ret) ret[(long long)i * a.ot] = A[i] + s.v[i];
    }
}

__device__ __forceinline__ int length_of(const Rollout& a, int n) {
    const int len = a.lengths ? a.lengths[n] : a.steps;
    return len < 0 ? 0 : len > a.steps ? a.steps : len;
}

// Steps before the first whole group of 4 in memory.
__device__ __forceinline__ int lead_of(const Rollout& a, int n) { return (int)((uintptr_t)(a.rewards + n * a.rn) / 4 % 4); }

// Lanes `apart` from one another hold consecutive steps: composes each with all after it within `width` lanes.
__device__ __forceinline__ Pair scan_lanes(Pair p, int apart, int width) {
    const int lane = threadIdx.x % width;
    for (int o = apart; o < width; o *= 2) {
        const Pair then{__shfl_down_sync(~0u, p.a, o, width), __shfl_down_sync(~0u, p.b, o, width)};
        if (lane + o < width) p = compose(p, then);
    }
    return p;
}

// Many environments, time consecutive in memory: `group` lanes an environment,
// 4 steps a lane, from the last steps to the first: 64 steps of 65,536
// environments 17 us, 256 of 16,384 17 us (the bytes alone 13).
constexpr int kRowThreads = 256;

template <class V, class D>
__global__ void __launch_bounds__(kRowThreads, 6) advantage_rows_kernel(const Rollout a, int group, int most_lead) {
    const long long place = ((long long)blockIdx.x * kRowThreads + threadIdx.x) / group;
    const bool on = place < a.envs;
    const int n = on ? (int)place : 0, lane = threadIdx.x % group;
    const int len = on ? length_of(a, n) : 0, lead = lead_of(a, n);
    // the same number of turns for a warp's environments
    const int turns = (a.steps + most_lead + 4 * group - 1) / (4 * group);
    float carry = 0.0f;
    for (int k = turns - 1; k >= 0; k--) {
        const int t = (k * group + lane) * 4 - lead;
        const Steps<4> s = load_steps<V, D, 4, true>(a, n, t, len);
        const Pair p = scan_lanes(s.pair(), 1, group);
        const Pair then{__shfl_down_sync(~0u, p.a, 1, group), __shfl_down_sync(~0u, p.b, 1, group)};
        if (on) store_steps<4, true>(a, s, n, t, len, lane == group - 1 ? carry : apply(then, carry));
        const Pair all{__shfl_sync(~0u, p.a, 0, group), __shfl_sync(~0u, p.b, 0, group)};
        carry = apply(all, carry);
    }
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ float remote_float(const void* p, unsigned rank) {
    unsigned at;
    float w;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(at) : "memory");
    return w;
}

constexpr int kMaxThreads = 1024;
constexpr int kBlockSteps = 8;   // steps a thread

constexpr int kMaxCluster = 8;

struct Shared {
    Pair total[2][kMaxThreads / 32][32];   // each warp's steps, by environment
    Pair block[32];                        // the block's
};

// 2^env_bits environments a block, neighbouring lanes neighbouring environments,
// kBlockSteps steps a thread; a cluster's blocks divide the time.  Long times take
// several turns of the block, from the last steps to the first, each with what
// the one before carried; the blocks of a cluster go through their part once
// before, for its pair alone (their second reading comes from L2).
//
// 64 steps of 4,096 environments side by side: 3.1 us, latency.  256 steps of
// 16,384: 18 us (4.7 TB/s, 73% of the copy rate).  1,024 environments of up to
// 8,191 steps one after the other, bf16 values: 34 us (68%), bound by the turns'
// chains of loads and joins at 64 registers a thread; loading a turn ahead took
// registers and 46 us (at 4 steps a thread, where this took 39).  65,536 steps
// of one environment: 13 us on a cluster's eight SMs.
template <class V, class D, bool kVec>
__global__ void __launch_bounds__(kMaxThreads) advantage_kernel(const Rollout a, int env_bits, int cluster) {
    constexpr int kSteps = kBlockSteps;
    __shared__ Shared sh;
    const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int nx = 1 << env_bits, e = threadIdx.x & (nx - 1), seg = threadIdx.x >> env_bits;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const long long place = (long long)(blockIdx.x / cluster) * nx + e;
    const bool on = place < a.envs;
    const int n = on ? (int)place : 0;
    const int len = on ? length_of(a, n) : 0;
    const int lead = kVec ? lead_of(a, n) : 0;
    const int turn = (blockDim.x >> env_bits) * kSteps;   // steps of a turn
    // this block's part of the time, from -lead on, in whole turns
    const int turns = (a.steps + lead + turn - 1) / turn, each = (turns + cluster - 1) / cluster;
    const int k0 = min(turns, each * rank), k1 = min(turns, k0 + each);

    int buffer = 0;
    Pair carry{1.0f, 0.0f};
    for (int phase = cluster > 1 ? 0 : 1; phase < 2; phase++) {
        for (int k = k1 - 1; k >= k0; k--) {
            const int t = k * turn + seg * kSteps - lead;
            const Steps<kSteps> s = load_steps<V, D, kSteps, kVec>(a, n, t, len);
            const Pair p = scan_lanes(s.pair(), nx, 32);
            if (lane < nx) sh.total[buffer][warp][lane] = p;
            __syncthreads();
            Pair here = carry;
            for (int w = warps - 1; w >= 0; w--) {
                if (w == warp) here = carry;
                carry = compose(sh.total[buffer][w][e], carry);
            }
            buffer ^= 1;
            if (phase == 0) continue;
            const Pair then{__shfl_down_sync(~0u, p.a, nx & 31), __shfl_down_sync(~0u, p.b, nx & 31)};
            if (on) store_steps<kSteps, kVec>(a, s, n, t, len, lane + nx >= 32 ? here.b : apply(then, here.b));
        }
        if (phase == 0) {
            if (threadIdx.x < nx) sh.block[threadIdx.x] = carry;
            cluster_sync();
            Pair after{1.0f, 0.0f};
            for (int r = cluster - 1; r > rank; r--)
                after = compose(Pair{remote_float(&sh.block[e].a, r), remote_float(&sh.block[e].b, r)}, after);
            carry = after;
            cluster_sync();   // no block leaves, or writes there, while another reads
        }
    }
}

template <class V, class D>
int launch(const Rollout& a, bool vec, cudaStream_t s) {
    const int lead = vec && ((uintptr_t)a.rewards % 16 || (a.envs > 1 && a.rn % 4)) ? 3 : 0;   // the most of any environment
    const int need = a.steps + lead;
    // Many environments, or few steps: lanes for each environment, no warp waits for another; 4 steps a lane (256 steps
    // of 16,384 environments 17 us, by blocks 24; 1,024 steps of 4,096 19 us, by blocks 18).
    if (vec && (a.steps <= 128 || a.envs >= 8192)) {
        int group = 1;
        while (group < 32 && group * 4 < need) group *= 2;
        const long long blocks = ((long long)a.envs * group + kRowThreads - 1) / kRowThreads;
        if (blocks > 0x7fffffff) return (int)cudaErrorInvalidValue;
        advantage_rows_kernel<V, D><<<(unsigned)blocks, kRowThreads, 0, s>>>(a, group, lead);
        return (int)cudaGetLastError();
    }
    // environments side by side where they are neighbours in memory, fewer while that leaves SMs idle and takes turns
    int bits = 0;
    if (!vec && (a.rt != 1 || a.steps == 1 || a.rn < a.rt)) {
        while (bits < 5 && (1 << bits) < a.envs) bits++;
        while (bits > 0 && ((a.envs + (1 << bits) - 1) >> bits) < 148 && a.steps > (kMaxThreads >> bits) * kBlockSteps) bits--;
    }
    const long long groups = ((long long)a.envs + (1 << bits) - 1) >> bits;
    // Threads for all steps, as many as suit (1,024 environments of 8,191 steps one after the other: 75 us with 512, 64
    // with 256, 34 with 128; 256 steps of 16,384 environments side by side: 20, 18, 22); all where blocks are few, and
    // clusters then (65,536 steps of one environment 13 us, by one block 44).
    const int most = groups < 148 ? kMaxThreads : vec ? 128 : 256;
    int threads = 32;
    while (threads < most && (threads >> bits) * kBlockSteps < need) threads *= 2;
    int cluster = 1;
    while (cluster < kMaxCluster && groups * cluster * 2 <= 148 && (long long)(threads >> bits) * kBlockSteps * cluster < need) cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(groups * cluster));
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    if (vec) return (int)cudaLaunchKernelEx(&cfg, advantage_kernel<V, D, true>, a, bits, cluster);
    return (int)cudaLaunchKernelEx(&cfg, advantage_kernel<V, D, false>, a, bits, cluster);
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
    if (!rewards || !values || !terminals || !last_values || !advantages || !strides || envs > (1ll << 30) ||
        steps > (1ll << 30) || (uintptr_t)rewards % 4 || (uintptr_t)values % vb || (uintptr_t)terminals % tb ||
        (uintptr_t)last_values % vb || (uintptr_t)lengths % 4 || (uintptr_t)advantages % 4 || (uintptr_t)returns % 4)
        return (int)cudaErrorInvalidValue;
    for (int i = 0; i < 11; i++)
        if (strides[i] < 0) return (int)cudaErrorInvalidValue;
    if (!apart(steps, envs, strides[7], strides[8]) || (returns && !apart(steps, envs, strides[9], strides[10])) ||
        (const void*)advantages == rewards || advantages == values || advantages == terminals || returns == advantages ||
        (returns && ((const void*)returns == rewards || returns == values || returns == terminals)))
        return (int)cudaErrorInvalidValue;
    const Rollout a{(int)steps, (int)envs, rewards, values, terminals, last_values, lengths, advantages, returns,
                    strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6],
                    strides[7], strides[8], strides[9], strides[10], gamma, gamma * lam != 0.0f ? gamma * lam : kCut};
    // 4 steps at a time: consecutive in memory, every array's rows at the same place among groups of 4
    const auto place = [](const void* p, int bytes) { return (uintptr_t)p / bytes % 4; };
    bool vec = steps > 1 && strides[0] == 1 && strides[2] == 1 && strides[4] == 1 && strides[7] == 1 &&
               (!returns || strides[9] == 1) && place(values, vb) == place(rewards, 4) &&
               place(terminals, tb) == place(rewards, 4) && place(advantages, 4) == place(rewards, 4) &&
               (!returns || place(returns, 4) == place(rewards, 4));
    if (envs > 1)
        for (const int i : {3, 5, 8, 10})
            vec = vec && ((!returns && i == 10) || (strides[i] - strides[1]) % 4 == 0);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool f = terminal_type == B3X_F32;
    if (value_type == B3X_F32) return f ? launch<float, float>(a, vec, s) : launch<float, unsigned char>(a, vec, s);
    if (value_type == B3X_BF16)
        return f ? launch<__nv_bfloat16, float>(a, vec, s) : launch<__nv_bfloat16, unsigned char>(a, vec, s);
    return f ? launch<__half, float>(a, vec, s) : launch<__half, unsigned char>(a, vec, s);
}
