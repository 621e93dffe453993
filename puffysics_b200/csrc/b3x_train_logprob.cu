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

// ---- ordered keys ---------------------------------------------------------------------
// Floats as whole numbers of the same order, both zeros as one.  NaN sorts above +infinity.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kNothing = 0x007FFFFFu;   // key_of(-infinity)
constexpr uint32_t kMost = 0xFF800000u;      // key_of(+infinity): NaN is above

// A logit and its index as one number: the larger logit, then the lower index, is larger.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t index) {
    return (uint64_t)key << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ int index_of(uint64_t e) { return (int)(0xFFFFFFFFu - (uint32_t)e); }

// ---- running sums -----------------------------------------------------------------------
// What a part of a row comes to: its maximum m, s = sum 2^x and t = sum x 2^x with
// x = c (z - m), c = scale log2 e.  Joined parts move to the larger maximum:
// 2^(x + d) (x + d) = 2^d (2^x x + d 2^x).  Exponents stop at -1e4, where 2^x is 0
// already, so that -infinity (d of an empty part, x of a masked logit) never
// meets a zero factor.  A NaN maximum stays; sums beside it mean nothing.
struct Part {
    float m, s, t;
};

__device__ __forceinline__ Part join(Part a, Part b, float c) {
    const float m = max_nan(a.m, b.m);
    const float da = fmaxf((a.m - m) * c, -1e4f), db = fmaxf((b.m - m) * c, -1e4f);
    const float fa = exp2_fast(da), fb = exp2_fast(db);
    return Part{m, a.s * fa + b.s * fb, __fmaf_rn(fa, __fmaf_rn(da, a.s, a.t), fb * __fmaf_rn(db, b.s, b.t))};
}

__device__ __forceinline__ Part join_lanes(Part a, float c, int lanes) {
    for (int o = lanes / 2; o; o >>= 1)
        a = join(a, Part{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)}, c);
    return a;
}

// A row's results from its sums.
struct Row {
    float m, logsum, entropy;
    __device__ __forceinline__ explicit Row(Part a) {
        const bool empty = a.m == -kInf;
        const float bad = empty ? 0.0f : a.m - a.m;   // NaN where the maximum is no number
        m = a.m;
        logsum = empty ? 0.0f : logf(a.s) + bad;
        entropy = empty ? 0.0f : logsum - 0.6931471805599453f * (a.t / a.s);
    }
    __device__ __forceinline__ float logp(float z, float scale) const {
        return z == -kInf && m == -kInf ? -kInf : (z - m) * scale - logsum;
    }
};

template <class T>
__device__ __forceinline__ void write_row(const Rows& a, const Out& o, long long row, const Row& r) {
    if (o.stats) o.stats[2 * row] = r.m, o.stats[2 * row + 1] = r.logsum;
    if (o.entropy) o.entropy[row] = r.entropy;
    if (o.logp) {
        const long long j = action_of(a, row);
        o.logp[row] = j >= 0 && j < a.width ? r.logp(logit<T>(a, row, (int)j), a.scale) : 0.0f;
    }
}

// ---- short rows -------------------------------------------------------------------------
// Up to 8 logits a lane, L lanes a row, all in registers: bound by latency and
// by the words a row has besides its logits.
constexpr int kShort = 8;
constexpr int kShortThreads = 256;

template <class T, int L>
__global__ void __launch_bounds__(kShortThreads) short_kernel(Rows a, Out o) {
    const long long row = ((long long)blockIdx.x * kShortThreads + threadIdx.x) / L;
    const int lane = threadIdx.x % L;
    const bool on = row < a.rows;
    float z[kShort];
    float m = -kInf;
#pragma unroll
    for (int i = 0; i < kShort; i++) {
        const int j = lane + i * L;
        z[i] = on && j < a.width ? logit<T>(a, row, j) : -kInf;
        m = max_nan(m, z[i]);
    }
    for (int k = L / 2; k; k >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, k));
    const float c = a.scale * kLog2e;
    Part p{m, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kShort; i++) {
        const float x = fmaxf((z[i] - m) * c, -1e4f), e = exp2_fast(x);
        p.s += e;
        p.t = __fmaf_rn(e, x, p.t);
    }
    for (int k = L / 2; k; k >>= 1) p.s += __shfl_xor_sync(~0u, p.s, k), p.t += __shfl_xor_sync(~0u, p.t, k);
    const Row r(p);
    if (on && lane == 0) write_row<T>(a, o, row, r);
    uint64_t last = ~0ull;
    for (int k = 0; k < o.top; k++) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < kShort; i++) {
            const uint32_t key = key_of(z[i]);
            const uint64_t e = entry_of(key, lane + i * L);
            if (key > kNothing && key <= kMost && e < last && e > best) best = e;
        }
        for (int q = L / 2; q; q >>= 1) {
            const uint64_t other = __shfl_xor_sync(~0u, best, q);
            best = other > best ? other : best;
        }
        last = best;
        if (on && lane == k % L) {
            const bool none = best == 0;
            o.top_ids[row * o.top + k] = none ? -1 : index_of(best);
            o.top_logp[row * o.top + k] = none ? -kInf : r.logp(of_key((uint32_t)(best >> 32)), a.scale);
        }
    }
}

// ---- long rows --------------------------------------------------------------------------
// 16 bytes of consecutive logits.  A row is cut on the 16-byte boundaries of
// memory, wherever it starts: vector v holds the elements from v N - head on.
template <class T> struct Vec { static constexpr int n = 16 / sizeof(T); };

__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 q;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
    return q;
}

template <class T> __device__ __forceinline__ uint32_t minus_infinity();
template <> __device__ __forceinline__ uint32_t minus_infinity<float>() { return 0xFF800000u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__nv_bfloat16>() { return 0xFF80FF80u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__half>() { return 0xFC00FC00u; }

// 0xFF in each byte that is not 0, as the sign bits of a word's bytes.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t x) { return ((x & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | x; }

template <class T, bool kMask>
struct Source {
    const T* row;
    const unsigned char* mask;
    int width, head;

    __device__ __forceinline__ Source(const Rows& a, long long r) {
        row = (const T*)a.logits + r * a.row_stride;
        mask = kMask ? a.mask + r * a.mask_stride : nullptr;
        width = a.width;
        head = (int)((uintptr_t)row % 16 / sizeof(T));
    }
    __device__ __forceinline__ int vectors() const { return (head + width + Vec<T>::n - 1) / Vec<T>::n; }

    // Vector v, -infinity where it is outside the row or masked.
    __device__ __forceinline__ uint4 load(int v) const {
        constexpr int N = Vec<T>::n;
        const int j = v * N - head;
        if (j >= 0 && j + N <= width) {
            uint4 q = load16(row + j);
            if (kMask) apply(q, j);
            return q;
        }
        uint32_t w[4] = {minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>()};
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (j + i < 0 || j + i >= width || (kMask && !mask[j + i])) continue;
            if (sizeof(T) == 4) w[i % 4] = reinterpret_cast<const uint32_t*>(row)[j + i];
            else {
                const uint32_t x = reinterpret_cast<const uint16_t*>(row)[j + i];
                w[i / 2 % 4] = i % 2 ? (w[i / 2 % 4] & 0xFFFFu) | x << 16 : (w[i / 2 % 4] & 0xFFFF0000u) | x;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }

    __device__ __forceinline__ void apply(uint4& q, int j) const {
        constexpr int N = Vec<T>::n;
        const unsigned char* p = mask + j;
        const int off = (int)((uintptr_t)p & 3);
        uint32_t b[2];
        // whole words around the N bytes, where they stay inside the row's own
        if (j >= off && j - off + N + 4 <= width) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(p - off);
            const uint32_t w0 = __ldg(w), w1 = N == 8 || off ? __ldg(w + 1) : 0u, w2 = N == 8 && off ? __ldg(w + 2) : 0u;
            b[0] = __funnelshift_r(w0, w1, off * 8);
            b[1] = __funnelshift_r(w1, w2, off * 8);
        } else {
            b[0] = b[1] = 0;
#pragma unroll
            for (int i = 0; i < N; i++) b[i / 4] |= (uint32_t)p[i] << i % 4 * 8;
        }
        uint32_t* w = &q.x;
        b[0] = nonzero_bytes(b[0]);
        if (N == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = b[0] >> i * 8 & 0x80u ? w[i] : minus_infinity<T>();
        } else {
            b[1] = nonzero_bytes(b[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) {   // a byte's sign bit becomes 16 bits of ones
                uint32_t keep;
                asm("prmt.b32 %0, %1, 0, %2;" : "=r"(keep) : "r"(b[i / 2]), "r"(i % 2 ? 0xBBAA : 0x9988));
                w[i] = (w[i] & keep) | (minus_infinity<T>() & ~keep);
            }
        }
    }
};

// The two logits of word i (one for float, the other -infinity).
template <class T> __device__ __forceinline__ float2 pair(uint32_t w);
template <> __device__ __forceinline__ float2 pair<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 pair<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// Element i of a vector.
template <class T> __device__ __forceinline__ float element(const uint4& q, int i) {
    const uint32_t* w = &q.x;
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else {
        const float2 f = pair<T>(w[i / 2]);
        return i % 2 ? f.y : f.x;
    }
}

template <class T> __device__ __forceinline__ float most(const uint4& q);
template <> __device__ __forceinline__ float most<float>(const uint4& q) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
}
template <> __device__ __forceinline__ float most<__nv_bfloat16>(const uint4& q) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 a = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(a), __high2float(a));
}
template <> __device__ __forceinline__ float most<__half>(const uint4& q) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    const __half2 a = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(a), __high2float(a));
}

// Two floats in one register pair, for the two-wide 32-bit arithmetic of sm_100.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

constexpr int kUnroll = 4;           // vectors a thread has in flight
constexpr int kGroups = 256;         // groups of consecutive vectors whose maxima are kept
constexpr int kFound = 512;          // logits at or above the threshold that are ranked at once
constexpr int kMaxWarps = 16;
constexpr int kMaxCluster = 8;

struct Shared {
    float m[kMaxWarps], s[kMaxWarps], t[kMaxWarps];
    Part part;                        // this block's
    Part joined;
    uint32_t group[kGroups];
    int order[B3X_TRAIN_MAX_TOP];
    uint32_t threshold;
    int found;
    uint64_t list[B3X_TRAIN_MAX_TOP]; // this block's alternatives
    uint64_t entries[kFound];
    uint64_t warp_best[kMaxWarps];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}
// A word of the same shared variable in another block of the cluster.
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
    uint32_t at, w;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
    return w;
}

// The K largest entries among the vectors of some groups (or all): each time
// the best one after the last.  Only for rows with many equal logits or NaN.
template <class T, bool kMask>
__device__ void search(const Source<T, kMask>& src, Shared& sh, int v0, int v1, int shift, const int* order, int groups,
                       int top) {
    const int warps = blockDim.x / 32;
    uint64_t last = ~0ull;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < groups << shift; i += blockDim.x) {
            const int v = v0 + (order ? (order[i >> shift] << shift) + (i & ((1 << shift) - 1)) : i);
            if (v >= v1) continue;
            const uint4 q = src.load(v);
            for (int n = 0; n < Vec<T>::n; n++) {
                const uint32_t key = key_of(element<T>(q, n));
                const uint64_t e = entry_of(key, v * Vec<T>::n - src.head + n);
                if (key > kNothing && key <= kMost && e < last && e > best) best = e;
            }
        }
        for (int o = 16; o; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(~0u, best, o);
            best = other > best ? other : best;
        }
        if (threadIdx.x % 32 == 0) sh.warp_best[threadIdx.x / 32] = best;
        __syncthreads();
        for (int w = 0; w < warps; w++) best = sh.warp_best[w] > best ? sh.warp_best[w] : best;
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) sh.list[k] = best;
    }
}

// The `top` largest of n entries (all different, none 0) in order, 0 beyond them.
__device__ __forceinline__ void rank_entries(const uint64_t* entries, int n, int top, uint64_t* list) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t e = entries[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += entries[j] > e;
        if (rank < top) list[rank] = e;
    }
    for (int i = n + threadIdx.x; i < top; i += blockDim.x) list[i] = 0;
}

// One block, or one cluster of blocks, a row.  Each warp takes kUnroll vectors a
// lane at a time and keeps the maximum, sum and weighted sum of each lane
// running; so a row is read once.  For the alternatives the maxima of groups of
// 2^shift consecutive vectors are kept beside.  The K groups with the largest
// maxima (the first among equal ones) hold the K largest logits, and the K-th of
// those maxima is at most the K-th largest logit: those groups are read again,
// from L2, and what reaches the threshold is ranked.
template <class T, bool kMask, bool kTop, int kThreads>
__global__ void __launch_bounds__(kThreads) long_kernel(Rows a, Out o, int cluster, int shift) {
    constexpr int N = Vec<T>::n;
    __shared__ Shared sh;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / cluster;
    const Source<T, kMask> src(a, row);
    const int nv = src.vectors();
    const int each = ((nv + cluster - 1) / cluster + (1 << shift) - 1) >> shift << shift;
    const int v0 = min(nv, each * rank), v1 = min(nv, v0 + each);
    const float c = a.scale * kLog2e;
    if (kTop) {
        for (int i = threadIdx.x; i < kGroups; i += blockDim.x) sh.group[i] = 0;
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
    }

    Part p{-kInf, 0.0f, 0.0f};
    for (int base = v0 + warp * 32 * kUnroll; base < v1; base += warps * 32 * kUnroll) {
        uint4 q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int v = base + u * 32 + lane;
            q[u] = make_uint4(minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>());
            if (v < v1) q[u] = src.load(v);
        }
        float top[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) top[u] = most<T>(q[u]);
        const float here = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        if (kTop) {
            if (shift >= 7) {
                const uint32_t key = __reduce_max_sync(~0u, key_of(here));
                if (lane == 0) atomicMax(&sh.group[(base - v0) >> shift], key);
            } else {
#pragma unroll
                for (int u = 0; u < kUnroll; u++) {
                    uint32_t key = key_of(top[u]);
                    for (int k = 0; k < shift; k++) key = max(key, __shfl_xor_sync(~0u, key, 1 << k));
                    const int v = base - v0 + u * 32 + lane;
                    if ((lane & ((1 << shift) - 1)) == 0 && v < v1 - v0) sh.group[v >> shift] = key;
                }
            }
        }
        const float m = max_nan(p.m, here);
        const float d = fmaxf((p.m - m) * c, -1e4f), f = exp2_fast(d);
        p = Part{m, p.s * f, f * __fmaf_rn(d, p.s, p.t)};
        const uint64_t minus = pack2(-m, -m), by = pack2(c, c);
        uint64_t s2 = 0, t2 = 0;
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const float2 z = make_float2(element<T>(q[u], 2 * i), element<T>(q[u], 2 * i + 1));
                float2 x = unpack2(mul2(add2(pack2(z.x, z.y), minus), by));
                x.x = fmaxf(x.x, -1e4f), x.y = fmaxf(x.y, -1e4f);
                const uint64_t e = pack2(exp2_fast(x.x), exp2_fast(x.y));
                s2 = add2(s2, e);
                t2 = fma2(e, pack2(x.x, x.y), t2);
            }
        }
        const float2 s = unpack2(s2), t = unpack2(t2);
        p.s += s.x + s.y;
        p.t += t.x + t.y;
    }
    p = join_lanes(p, c, 32);
    if (lane == 0) sh.m[warp] = p.m, sh.s[warp] = p.s, sh.t[warp] = p.t;
    __syncthreads();
    p = Part{sh.m[0], sh.s[0], sh.t[0]};
    for (int w = 1; w < warps; w++) p = join(p, Part{sh.m[w], sh.s[w], sh.t[w]}, c);

    if (kTop) {
        const int groups = (v1 - v0 + (1 << shift) - 1) >> shift;
        if (p.m != p.m) {
            search<T, kMask>(src, sh, v0, v1, shift, nullptr, groups, o.top);
        } else {
            const int chosen = min(o.top, groups);
            for (int g = threadIdx.x; g < groups; g += blockDim.x) {
                const uint32_t key = sh.group[g];
                int above = 0;
                for (int k = 0; k < groups; k++) above += sh.group[k] > key || (sh.group[k] == key && k < g);
                if (above < chosen) sh.order[above] = g;
                if (above == o.top - 1) sh.threshold = key;
            }
            if (groups < o.top && threadIdx.x == 0) sh.threshold = 0;
            __syncthreads();
            const uint32_t threshold = max(sh.threshold, kNothing + 1);
            for (int i = threadIdx.x; i < chosen << shift; i += blockDim.x) {
                const int v = v0 + (sh.order[i >> shift] << shift) + (i & ((1 << shift) - 1));
                if (v >= v1) continue;
                const uint4 q = src.load(v);
                if (key_of(most<T>(q)) < threshold) continue;
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const uint32_t key = key_of(element<T>(q, n));
                    if (key < threshold) continue;
                    const int at = atomicAdd(&sh.found, 1);
                    if (at < kFound) sh.entries[at] = entry_of(key, v * N - src.head + n);
                }
            }
            __syncthreads();
            const int found = sh.found;
            if (found <= kFound) rank_entries(sh.entries, found, o.top, sh.list);
            else search<T, kMask>(src, sh, v0, v1, shift, sh.order, chosen, o.top);
        }
        __syncthreads();
    }

    if (cluster > 1) {
        if (threadIdx.x == 0) sh.part = p;
        cluster_sync();
        if (rank == 0) {
            for (int r = 1; r < cluster; r++)
                p = join(p, Part{__uint_as_float(remote(&sh.part.m, r)), __uint_as_float(remote(&sh.part.s, r)),
                                 __uint_as_float(remote(&sh.part.t, r))}, c);
            if (kTop) {
                if (threadIdx.x == 0) sh.found = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < cluster * o.top; i += blockDim.x) {
                    const uint64_t* at = &sh.list[i % o.top];
                    const uint64_t e = (uint64_t)remote((const char*)at + 4, i / o.top) << 32 | remote(at, i / o.top);
                    if (e) sh.entries[atomicAdd(&sh.found, 1)] = e;
                }
                __syncthreads();
                rank_entries(sh.entries, sh.found, o.top, sh.list);
                __syncthreads();
            }
        }
        cluster_sync();   // no block leaves while its shared memory is read
        if (rank) return;
    }
    const Row r(p);
    if (threadIdx.x == 0) write_row<T>(a, o, row, r);
    if (kTop)
        for (int k = threadIdx.x; k < o.top; k += blockDim.x) {
            const uint64_t e = sh.list[k];
            o.top_ids[row * o.top + k] = e ? index_of(e) : -1;
            o.top_logp[row * o.top + k] = e ? r.logp(of_key((uint32_t)(e >> 32)), a.scale) : -kInf;
        }
}
static_assert(kMaxCluster * B3X_TRAIN_MAX_TOP <= kFound, "the blocks' alternatives are ranked at once");

template <class T, int L>
int launch_short(const Rows& a, const Out& o, cudaStream_t s) {
    const long long per = kShortThreads / L;
    short_kernel<T, L><<<(unsigned)((a.rows + per - 1) / per), kShortThreads, 0, s>>>(a, o);
    return (int)cudaGetLastError();
}

template <class T, bool kMask, bool kTop>
int launch_long(const Rows& a, const Out& o, cudaStream_t s) {
    const int nv = (int)(((long long)a.width + Vec<T>::n - 1) / Vec<T>::n) + 1;
    // a cluster a row while rows alone leave SMs idle and each block keeps 512 vectors
    int cluster = 1;
    while (cluster < kMaxCluster && a.rows * cluster * 2 <= 296 && nv / (cluster * 2) >= 512) cluster *= 2;
    const int each = (nv + cluster - 1) / cluster;
    int warps = 1;
    while (warps < kMaxWarps && warps * 32 * kUnroll < each) warps *= 2;
    int shift = 0;
    while ((each + (1 << shift) - 1) >> shift > kGroups) shift++;
    if (shift == 6) shift = 7;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * cluster));
    cfg.blockDim = dim3(warps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, long_kernel<T, kMask, kTop, kMaxWarps * 32>, a, o, cluster, shift);
}

template <class T>
int launch(const Rows& a, const Out& o, cudaStream_t s) {
    if (a.width <= kShort) return launch_short<T, 1>(a, o, s);
    if (a.width <= kShort * 2) return launch_short<T, 2>(a, o, s);
    if (a.width <= kShort * 4) return launch_short<T, 4>(a, o, s);
    if (a.width <= kShort * 8) return launch_short<T, 8>(a, o, s);
    if (a.width <= kShort * 16) return launch_short<T, 16>(a, o, s);
    if (a.width <= kShort * 32) return launch_short<T, 32>(a, o, s);
    if (a.mask) return o.top ? launch_long<T, true, true>(a, o, s) : launch_long<T, true, false>(a, o, s);
    return o.top ? launch_long<T, false, true>(a, o, s) : launch_long<T, false, false>(a, o, s);
}

struct Grad {
    const float *stats, *entropy, *d_logp, *d_entropy;
    void* grad;
    long long grad_stride;
};

constexpr int kThreads = 256;

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
    if (type == B3X_F32) return launch<float>(a, o, (cudaStream_t)stream);
    if (type == B3X_BF16) return launch<__nv_bfloat16>(a, o, (cudaStream_t)stream);
    return launch<__half>(a, o, (cudaStream_t)stream);
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
