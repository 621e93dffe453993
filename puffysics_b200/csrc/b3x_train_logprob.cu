// b3x_train_logprob.cu -- log probabilities of actions, entropies and most
// likely alternatives of rows of logits (b3x_train.h).
#include <type_traits>

#include "b3x_train_rows.cuh"

using namespace b3t;

namespace {

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

// scale log2 e, within the floats for any finite scale: from 2.4e38 on only a
// row's maximum has a probability, with that factor as with the largest float.
__device__ __forceinline__ float factor_of(const Rows& a) { return fminf(a.scale * kLog2e, 3.402823466e38f); }

// ---- running sums -----------------------------------------------------------------------
// What a part of a row comes to: its maximum m, a whole number r near c m
// (c = scale log2 e), s = sum 2^x and t = sum x 2^x with x = c z - r.  r is
// exact, so one fused operation gives x with a rounding of its own size only,
// and what c's rounding does to c z it does to c m as well:
//   L = ln s - ln 2 (c m - r),  H = ln s - ln 2 t / s.
// Joined parts move to the larger r: 2^(x + d) (x + d) = 2^d (2^x x + d 2^x).
// Shifts and exponents stop at -1e4, where 2^x is 0 already, so that -infinity
// never meets a zero factor.  From |c m| = 2^24 on, whole numbers that floats
// hold are not always near c m: a row whose maximum has none is summed about the
// maximum itself, and a part of such logits (a stretch filled with -1e9, say), whose
// sums may be beyond the floats, is dropped where 2^d is 0: in any other row it
// weighs nothing.  A NaN maximum stays; sums beside it mean nothing.
struct Part {
    float m, r, s, t;
};
__device__ __forceinline__ Part empty_part() { return Part{-kInf, -3.0e38f, 0.0f, 0.0f}; }

__device__ __forceinline__ float reference(float m, float c) { return fminf(fmaxf(rintf(m * c), -3.0e38f), 3.0e38f); }

__device__ __forceinline__ Part moved(Part a, float m, float r) {
    const float d = fmaxf(a.r - r, -1e4f), f = exp2_fast(d);
    if (f == 0.0f) return Part{m, r, 0.0f, 0.0f};   // its sums may be beyond the floats
    return Part{m, r, a.s * f, f * __fmaf_rn(d, a.s, a.t)};
}

// A warp's maximum, keeping a NaN.
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ Part join_lanes(Part a) {
    a = moved(a, warp_max(a.m), warp_max(a.r));
    for (int o = 16; o; o >>= 1) a.s += __shfl_xor_sync(~0u, a.s, o), a.t += __shfl_xor_sync(~0u, a.t, o);
    return a;
}

// Whether no whole number is near enough to c m (possible from 2^24 on): the row
// needs sums of (z - m) instead.  Up to 40 above r the sums lose nothing but what
// ln s and ln 2 t / s, of up to 28 each, cost the entropy in their last places;
// below r by more than 2 a dropped part could weigh something.
__device__ __forceinline__ bool out_of_range(const Part& a, float c) {
    const float x = __fmaf_rn(a.m, c, -a.r);
    return fabsf(a.m) < kInf && !(x >= -2.0f && x <= 40.0f);
}

constexpr float kLn2 = 0.6931471805599453f;

// A row's results from its sums.
struct Row {
    float m, logsum, entropy;
    __device__ __forceinline__ Row(Part a, float c) {
        const bool empty = a.m == -kInf;
        const float bad = empty ? 0.0f : a.m - a.m;   // NaN where the maximum is no number
        m = a.m;
        const float log_s = logf(a.s);
        logsum = empty ? 0.0f : __fmaf_rn(-kLn2, __fmaf_rn(a.m, c, -a.r), log_s) + bad;
        entropy = empty ? 0.0f : __fmaf_rn(-kLn2, a.t / a.s, log_s) + bad;
    }
    // The same where x was c (z - m): r is c m itself.
    static __device__ __forceinline__ Row about_maximum(Part a) {
        a.r = 0.0f;
        const float m = a.m;
        a.m = m == -kInf || m - m != 0.0f ? m : 0.0f;
        Row row(a, 0.0f);
        row.m = m;
        return row;
    }
    __device__ __forceinline__ float logp(float z, float scale) const {
        return z == -kInf && m == -kInf ? -kInf : (z - m) * scale - logsum;
    }
};

// A row's action, read ahead of the sums.
struct Action {
    bool any;
    float z;
};
template <class T>
__device__ __forceinline__ Action load_action(const Rows& a, const Out& o, long long row) {
    Action got{false, 0.0f};
    if (o.logp) {
        const long long j = action_of(a, row);
        got.any = j >= 0 && j < a.width;
        if (got.any) got.z = logit<T>(a, row, (int)j);
    }
    return got;
}

__device__ __forceinline__ void write_row(const Rows& a, const Out& o, long long row, const Row& r, Action act) {
    if (o.stats) o.stats[2 * row] = r.m, o.stats[2 * row + 1] = r.logsum;
    if (o.entropy) o.entropy[row] = r.entropy;
    if (o.logp) o.logp[row] = act.any ? r.logp(act.z, a.scale) : 0.0f;
}

__device__ __forceinline__ void write_top(const Out& o, long long row, int k, uint64_t e, const Row& r, float scale) {
    o.top_ids[row * o.top + k] = e ? index_of(e) : -1;
    o.top_logp[row * o.top + k] = e ? r.logp(of_key((uint32_t)(e >> 32)), scale) : -kInf;
}

// ---- rows of a thread ---------------------------------------------------------------------
// Up to 8 logits, one thread a row, all in registers: bound by the launch and by
// the words that a row has besides its logits (4,096 rows of 3: 1.8 us).
constexpr int kShort = 8;
constexpr int kShortThreads = 128;

template <class T>
__global__ void __launch_bounds__(kShortThreads) short_kernel(Rows a, Out o) {
    const long long row = (long long)blockIdx.x * kShortThreads + threadIdx.x;
    if (row >= a.rows) return;
    const Action act = load_action<T>(a, o, row);
    float z[kShort];
    Part p{-kInf, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kShort; i++) {
        z[i] = i < a.width ? logit<T>(a, row, i) : -kInf;
        p.m = max_nan(p.m, z[i]);
    }
    const float c = factor_of(a);
#pragma unroll
    for (int i = 0; i < kShort; i++) {   // the maximum is known before the sums: x = c (z - m)
        const float x = fmaxf((z[i] - p.m) * c, -1e4f), e = exp2_fast(x);
        p.s += e;
        p.t = __fmaf_rn(e, x, p.t);
    }
    const Row r = Row::about_maximum(p);
    write_row(a, o, row, r, act);
    uint64_t last = ~0ull;
    for (int k = 0; k < o.top; k++) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < kShort; i++) {
            const uint32_t key = key_of(z[i]);
            const uint64_t e = entry_of(key, i);
            if (key > kNothing && key <= kMost && e < last && e > best) best = e;
        }
        last = best;
        write_top(o, row, k, best, r, a.scale);
    }
}

// U vectors' part of s and t.  What is -infinity is known only by the NaN it
// leaves in t (0 times -infinity): then, and always with a mask, once more with
// the exponents stopped, which costs an instruction a logit.
template <class T, int U, bool kMask>
__device__ __forceinline__ void add_vectors(const uint4 (&q)[U], float c, Part& p) {
    constexpr int N = Vec<T>::n;
    const uint64_t by = pack2(c, c), minus = pack2(-p.r, -p.r);
    uint64_t s2, t2;
    auto go = [&](bool stop) {
        s2 = t2 = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                float2 x = unpack2(fma2(pack2(element<T>(q[u], 2 * i), element<T>(q[u], 2 * i + 1)), by, minus));
                if (stop) x.x = fmaxf(x.x, -1e4f), x.y = fmaxf(x.y, -1e4f);
                const uint64_t e = pack2(exp2_fast(x.x), exp2_fast(x.y));
                s2 = add2(s2, e);
                t2 = fma2(e, pack2(x.x, x.y), t2);
            }
        }
    };
    go(kMask);
    float2 t = unpack2(t2);
    if (!kMask && t.x + t.y != t.x + t.y) {
        go(true);
        t = unpack2(t2);
    }
    const float2 s = unpack2(s2);
    p.s += s.x + s.y;
    p.t += t.x + t.y;
}

template <class T, int U>
__device__ __forceinline__ float most_of(const uint4 (&q)[U]) {
    float m = most<T>(q[0]);
#pragma unroll
    for (int u = 1; u < U; u++) m = max_nan(m, most<T>(q[u]));
    return m;
}

// The lanes' keys from the largest down.
__device__ __forceinline__ uint32_t sort_lanes(uint32_t key) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int j = k / 2; j; j /= 2) {
            const uint32_t other = __shfl_xor_sync(~0u, key, j);
            const bool larger = ((lane & j) == 0) == ((lane & k) == 0);
            key = larger ? max(key, other) : min(key, other);
        }
    return key;
}

// The 32 largest of two sorted lists, sorted: the larger of each key and its
// mirror image rise and fall once.
__device__ __forceinline__ uint32_t merge_lanes(uint32_t key, uint32_t mirrored) {
    const int lane = threadIdx.x % 32;
    key = max(key, mirrored);
#pragma unroll
    for (int j = 16; j; j /= 2) {
        const uint32_t other = __shfl_xor_sync(~0u, key, j);
        key = (lane & j) == 0 ? max(key, other) : min(key, other);
    }
    return key;
}

// Of a warp's 32 vectors from v on (those before v1) the logits with this key, in
// order, as entries from out[got] on, no more than `need` in all; how many there are then.
template <class T, class S>
__device__ __forceinline__ int take_equal(const S& src, int v, int v1, uint32_t key, uint64_t* out, int need, int got) {
    constexpr int N = Vec<T>::n;
    v += threadIdx.x % 32;
    const uint4 q = v < v1 ? src.load(v) : no_vector<T>();
    uint32_t bits = 0;
#pragma unroll
    for (int n = 0; n < N; n++) bits |= key_of(element<T>(q, n)) == key ? 1u << n : 0;
    int at = __popc(bits);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int before = __shfl_up_sync(~0u, at, o);
        if (threadIdx.x % 32 >= o) at += before;
    }
    const int all = __shfl_sync(~0u, at, 31);
    at += got - __popc(bits);
    while (bits && at < need) {
        out[at++] = entry_of(key, v * N - src.head + __ffs(bits) - 1);
        bits &= bits - 1;
    }
    return min(need, got + all);
}

// The sums of a row that is out of range: x = c (z - m).  `by`: threads that
// share the row.
template <class T, bool kMask>
__device__ __noinline__ float2 far_sums(const Source<T, kMask>& src, float m, float c, int first, int by) {
    float s = 0.0f, t = 0.0f;
    for (int v = first; v < src.vectors(); v += by) {
        const uint4 q = src.load(v);
        for (int n = 0; n < Vec<T>::n; n++) {
            const float x = fmaxf((element<T>(q, n) - m) * c, -1e4f), e = exp2_fast(x);
            s += e;
            t = __fmaf_rn(e, x, t);
        }
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o), t += __shfl_xor_sync(~0u, t, o);
    return make_float2(s, t);
}

// ---- rows of some lanes -------------------------------------------------------------------
// Rows of up to 4 L vectors, L lanes a row, in registers.  Or (kWalk, 32 lanes)
// of more, which the warp walks over twice when alternatives are asked for, the
// second time from L2.
//
// Alternatives: a threshold that K logits reach, then what reaches it is ranked.
// With 32 lanes it is the K-th largest of the lanes' maxima, with fewer that of
// the vectors'; where there are fewer vectors than alternatives it is no
// threshold at all.  A row has room for 8 candidates a lane.  More than that
// takes K passes over the row, and it is the rule, not the exception, with more
// alternatives than vectors (16-bit rows of 17 to 128 logits with 20, of 17 to
// 256 with 32) as with 29 and more of 32 maxima, which some 70 to 130 logits
// reach: 65,536 bf16 rows of 50 logits with 20 alternatives 106 us, of 100 183
// us, of 200 61 us and with 32 alternatives 468 us, of 1,000 with 32 384 us.
//
// Lanes by the row's length, so that a lane has up to 4 vectors in flight and the
// reductions and a row's last steps (a logarithm, a division, its stores) are
// shared by as few as will do.  Bound by issued instructions and by latency, not
// by memory: 147,456 masked rows of 21 f32 with the greedy action 8.5 us (the
// bytes alone 3.1), 65,536 rows of 1,000 bf16 45 us (20.6), with 20 alternatives
// 104.  Without alternatives five blocks an SM (four 49 us); with them four.
// At 48 and 64 registers a thread the 16-bit forms spill: up to 40 bytes without
// alternatives, 96 to 144 with them.
constexpr int kRowThreads = 256;
constexpr int kRowFound = 256;       // logits that are ranked at once, for a warp's rows together

// A bit for each logit of U vectors that reaches z: bit 4 u + i for word i of
// vector u, and from bit 16 on for the words' upper halves.
template <class T, int U>
__device__ __forceinline__ uint32_t reach(const uint4 (&q)[U], float z) {
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t* w = &q[u].x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t one = 0x00010001u << (u * 4 + i);
            if constexpr (sizeof(T) == 4) {
                if (__uint_as_float(w[i]) >= z) bits |= one & 0xFFFFu;
            } else if constexpr (sizeof(T) == 2 && Vec<T>::n == 8) {
                uint32_t m;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) m = __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), __float2bfloat162_rn(z));
                else m = __hge2_mask(*reinterpret_cast<const __half2*>(&w[i]), __float2half2_rn(z));
                bits |= m & one;
            }
        }
    }
    return bits;
}

// The lowest value of type T: what -infinity does not reach.
template <class T> __device__ __forceinline__ float lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ float lowest<__nv_bfloat16>() { return __uint_as_float(0xFF7F0000u); }
template <> __device__ __forceinline__ float lowest<__half>() { return -65504.0f; }


template <class T, bool kMask, bool kTop, int L, bool kWalk>
__global__ void __launch_bounds__(kRowThreads, kTop ? 4 : 5) lanes_kernel(Rows a, Out o) {
    constexpr int N = Vec<T>::n, U = 4, kRows = 32 / L, kCap = kRowFound / kRows, kFew = L == 32 ? 96 : kCap;
    __shared__ uint64_t entries[kTop ? kRowThreads / L : 1][kTop ? kCap : 1];
    __shared__ __align__(16) uint32_t best[kTop && L < 32 ? kRowThreads / L : 1][kTop && L < 32 ? U * L : 1];
    __shared__ int found[kTop ? kRowThreads / L : 1];
    const int here = threadIdx.x / L, lane = threadIdx.x % L;
    const long long row = (long long)blockIdx.x * (kRowThreads / L) + here;
    const bool on = row < a.rows;
    const Source<T, kMask, kTop> src(a, on ? row : 0);
    const int nv = on ? src.vectors() : 0;
    const float c = factor_of(a);
    if (kTop && lane == 0) found[here] = 0;
    Action act{false, 0.0f};
    if (on && lane == 0) act = load_action<T>(a, o, row);
    uint4 q[U];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = base + u * L + lane;
            q[u] = v < nv ? src.load(v) : no_vector<T>();
        }
    };
    Part p = empty_part();
    float mine = -kInf;
    if (kWalk) {
        for (int base = 0; base < nv; base += U * L) {
            if (base >= 2 && base + U * L <= src.last()) {
#pragma unroll
                for (int u = 0; u < U; u++) q[u] = src.inner(base + u * L + lane);
            } else {
                load(base);
            }
            const float m = max_nan(p.m, most_of<T, U>(q));
            p = moved(p, m, reference(m, c));
            add_vectors<T, U, kMask>(q, c, p);
        }
        mine = p.m;
        p = join_lanes(p);
    } else {
        load(0);
        p.m = mine = most_of<T, U>(q);
#pragma unroll
        for (int k = L / 2; k; k /= 2) p.m = max_nan(p.m, __shfl_xor_sync(~0u, p.m, k));
        p.r = reference(p.m, c);
        add_vectors<T, U, kMask>(q, c, p);
#pragma unroll
        for (int k = L / 2; k; k /= 2) p.s += __shfl_xor_sync(~0u, p.s, k), p.t += __shfl_xor_sync(~0u, p.t, k);
    }
    const bool far = out_of_range(p, c);
    if (__any_sync(~0u, far)) {   // x = c (z - m)
        float s = 0.0f, t = 0.0f;
        for (int v = lane; v < nv; v += L) {
            const uint4 w = src.load(v);
            for (int n = 0; n < N; n++) {
                const float x = fmaxf((element<T>(w, n) - p.m) * c, -1e4f), e = exp2_fast(x);
                s += e;
                t = __fmaf_rn(e, x, t);
            }
        }
        for (int k = L / 2; k; k /= 2) s += __shfl_xor_sync(~0u, s, k), t += __shfl_xor_sync(~0u, t, k);
        if (far) p.s = s, p.t = t;
    }
    const Row r = far ? Row::about_maximum(p) : Row(p, c);
    if (on && lane == 0) write_row(a, o, row, r, act);
    if (!kTop) return;

    if (!kWalk && o.top == 1 && __all_sync(~0u, p.m == p.m)) {   // the first place of the maximum
        int first = 0x7FFFFFFF;
#pragma unroll
        for (int u = U - 1; u >= 0; u--)
#pragma unroll
            for (int n = N - 1; n >= 0; n--)
                if (element<T>(q[u], n) == p.m) first = (u * L + lane) * N - src.head + n;
#pragma unroll
        for (int k = L / 2; k; k /= 2) first = min(first, __shfl_xor_sync(~0u, first, k));
        if (on && lane == 0) write_top(o, row, 0, p.m == -kInf ? 0 : entry_of(key_of(p.m), first), r, a.scale);
        return;
    }

    float z;
    if (L == 32) {
        z = of_key(__shfl_sync(~0u, sort_lanes(key_of(mine)), o.top - 1));
    } else {
        uint32_t key[U];
#pragma unroll
        for (int u = 0; u < U; u++) best[here][u * L + lane] = key[u] = key_of(most<T>(q[u]));
        __syncwarp();
        int above[U] = {};
        const uint4* all = reinterpret_cast<const uint4*>(best[here]);
        for (int i = 0; i < U * L / 4; i++) {
            const uint4 w = all[i];
#pragma unroll
            for (int u = 0; u < U; u++) above[u] += (w.x > key[u]) + (w.y > key[u]) + (w.z > key[u]) + (w.w > key[u]);
        }
        // the least of those that fewer than K are above
#pragma unroll
        for (int u = 0; u < U; u++)
            if (above[u] >= o.top) key[u] = ~0u;
        uint32_t least = min(min(key[0], key[1]), min(key[2], key[3]));
#pragma unroll
        for (int k = L / 2; k; k /= 2) least = min(least, __shfl_xor_sync(~0u, least, k));
        z = o.top <= U * L ? of_key(least) : -kInf;   // too few vectors: every logit
    }
    z = fmaxf(z, lowest<T>());
    __syncwarp();
    for (int base = 0; base < (kWalk ? nv : 1); base += U * L) {
        if (kWalk) load(base);
        uint32_t bits = reach<T, U>(q, z);
        if (bits) {
            int at = atomicAdd(&found[here], __popc(bits));
            while (bits) {
                const int b = __ffs(bits) - 1, w = b & 15;
                bits &= bits - 1;
                if (at < kCap) entries[here][at] = (base + (w >> 2) * L + lane) * N - src.head + (w & 3) * (N / 4) + (b >> 4);
                at++;
            }
        }
    }
    __syncwarp();
    int n = found[here];
    bool ranked = n <= kFew && p.m == p.m;
    if (ranked) {
        for (int i = lane; i < n; i += L) {
            const int j = (int)entries[here][i];
            entries[here][i] = entry_of(key_of(to_float(src.row[j])), j);
        }
    } else if (L == 32 && p.m == p.m) {
        // more than are ranked at once, as where many are equal to the threshold and with 31 or 32 alternatives: all above
        // it, then the first of those that are equal to it
        const uint32_t key = key_of(z);
        __syncwarp();
        if (lane == 0) found[here] = 0;
        __syncwarp();
        for (int v = lane; v < nv; v += 32) {
            const uint4 x = src.load(v);
            if (key_of(most<T>(x)) <= key) continue;
            for (int i = 0; i < N; i++) {
                const uint32_t k = key_of(element<T>(x, i));
                if (k <= key) continue;
                const int at = atomicAdd(&found[here], 1);
                if (at >= kCap) break;
                entries[here][at] = entry_of(k, v * N - src.head + i);
            }
        }
        __syncwarp();
        n = found[here];
        for (int v = 0; v < nv && n < o.top; v += 32) n = take_equal<T>(src, v, nv, key, entries[here], o.top, n);
        ranked = n <= kCap;
    }
    __syncwarp();
    if (ranked && on) {
        for (int i = lane; i < n; i += L) {
            const uint64_t e = entries[here][i];
            int rank = 0;
            for (int j = 0; j < n; j++) rank += entries[here][j] > e;
            if (rank < o.top) write_top(o, row, rank, e, r, a.scale);
        }
        for (int i = n + lane; i < o.top; i += L) write_top(o, row, i, 0, r, a.scale);
    }
    if (__all_sync(~0u, ranked)) return;
    // more logits than there is room for, or NaN: each time the best one after the last
    uint64_t last = ~0ull;
    for (int k = 0; k < o.top; k++) {
        uint64_t top = 0;
        for (int v = lane; v < nv; v += L) {
            const uint4 x = src.load(v);
            for (int i = 0; i < N; i++) {
                const uint32_t key = key_of(element<T>(x, i));
                const uint64_t e = entry_of(key, v * N - src.head + i);
                if (key > kNothing && key <= kMost && e < last && e > top) top = e;
            }
        }
        for (int d = L / 2; d; d /= 2) {
            const uint64_t other = __shfl_xor_sync(~0u, top, d);
            top = other > top ? other : top;
        }
        last = top;
        if (on && !ranked && lane == 0) write_top(o, row, k, top, r, a.scale);
    }
}

// ---- rows of a block or a cluster ------------------------------------------------------------
constexpr int kUnroll = 4;           // vectors a thread has in flight
constexpr int kTile = 32 * kUnroll;  // vectors a warp takes at a time
constexpr int kGroups = 512;         // groups of consecutive vectors whose maxima are kept
constexpr int kFound = 256;          // logits at or above the threshold that are ranked at once
constexpr int kMaxWarps = 16;
constexpr int kMaxCluster = 8;
constexpr int kSmallWarps = 4, kSmallBlocks = 8;   // of a block where there are many rows

struct Shared {
    Part part[kMaxWarps];
    Part all;                         // this block's
    uint32_t group[kGroups];
    uint32_t sorted[kMaxWarps][32];   // the lanes' maxima
    int order[kGroups];
    int chosen, found;
    uint64_t list[B3X_TRAIN_MAX_TOP]; // this block's alternatives
    uint64_t joined[B3X_TRAIN_MAX_TOP];
    uint64_t entries[kFound];
    uint64_t warp_best[kMaxWarps];
    float2 far[kMaxWarps];
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
__device__ __forceinline__ float remote_float(const void* p, uint32_t rank) { return __uint_as_float(remote(p, rank)); }

// The K largest entries among the vectors of some groups (or all): each time
// the best one after the last.  Only for rows with NaN, or with more logits above
// the threshold than are ranked at once.
template <class T, bool kMask>
__device__ __noinline__ void search(const Source<T, kMask>& src, Shared& sh, int v0, int v1, int shift, const int* order,
                                    int groups, int top) {
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
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += entries[j] > e;
        if (rank < top) list[rank] = e;
    }
    for (int i = n + threadIdx.x; i < top; i += blockDim.x) list[i] = 0;
}

// Adds a vector's logits that reach the threshold to the entries.
template <class T, bool kMask>
__device__ __forceinline__ void gather(const Source<T, kMask>& src, Shared& sh, const uint4& q, int v, uint32_t threshold) {
    if (key_of(most<T>(q)) < threshold) return;
#pragma unroll
    for (int n = 0; n < Vec<T>::n; n++) {
        const uint32_t key = key_of(element<T>(q, n));
        if (key < threshold) continue;
        const int at = atomicAdd(&sh.found, 1);
        if (at >= kFound) return;   // too many to rank already
        sh.entries[at] = entry_of(key, v * Vec<T>::n - src.head + n);
    }
}

// The `top` groups with the largest maxima, the first among equal ones: they hold the `top` largest logits.
__device__ __noinline__ void best_groups(Shared& sh, int groups, int top) {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        const uint32_t key = sh.group[g];
        int above = 0;
        for (int k = 0; k < groups; k++) above += sh.group[k] > key || (sh.group[k] == key && k < g);
        if (above < top) sh.order[above] = g;
    }
    __syncthreads();
}

// The alternatives of a row with more logits at the threshold than are ranked at
// once, by far the most equal to it: all above it, then the first of those.
template <class T, bool kMask, bool kOnce>
__device__ __noinline__ void crowded(const Source<T, kMask>& src, Shared& sh, int v0, int v1, int shift, int groups, int top,
                                     uint32_t threshold) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (int v = v0 + threadIdx.x; v < v1; v += blockDim.x)
        if (kOnce || sh.group[(v - v0) >> shift] > threshold) gather(src, sh, src.load(v), v, threshold + 1);
    __syncthreads();
    if (threadIdx.x < 32 && sh.found < top) {
        int n = sh.found;
        for (int v = v0; v < v1 && n < top; v += 32)
            if (kOnce || sh.group[(v - v0) >> shift] >= threshold) n = take_equal<T>(src, v, v1, threshold, sh.entries, top, n);
        if (threadIdx.x == 0) sh.found = n;
    }
    __syncthreads();
    const int found = sh.found;
    if (found <= kFound) {
        rank_entries(sh.entries, found, top, sh.list);
    } else if (kOnce) {
        search<T, kMask>(src, sh, v0, v1, 0, nullptr, v1 - v0, top);
    } else {
        best_groups(sh, groups, top);
        search<T, kMask>(src, sh, v0, v1, shift, sh.order, min(top, groups), top);
    }
}

// One block, or one cluster of blocks, a row; the row is read once.  kOnce: each
// warp has one tile, which stays in its registers.  Otherwise the warps walk
// over the row with their sums running.
//
// Alternatives.  The lanes' maxima are sorted by warps and merged: the K-th of
// them is at most the K-th largest logit.  What reaches it is ranked: from the
// registers, or, where the row was walked over, from the groups of 2^shift
// consecutive vectors whose maxima (kept beside) reach it, which are read again
// from L2.
//
// 4,096 rows of 131,072 bf16: 177 us without alternatives (6.1 TB/s, 94% of the
// copy rate), 215 to 219 with 20 (77%).  An exponential a logit keeps the special
// function unit half busy; the rest of the time is the loads' latency at 64
// registers a thread, and each row's end (sorting, ranking), which other blocks
// of the SM cover in part.  12 blocks an SM instead of 8 spill (267 us).  8 rows,
// a cluster of 8 blocks each: 4.7 us without alternatives, 9.7 with 20, all of it
// latency; kOnce with alternatives spills 100 bytes a thread at 64 registers.  Rows
// that are out of range are read a second time (4,096 rows all of -1e10: 488 us).
template <class T, bool kMask, bool kTop, bool kOnce, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == kMaxWarps ? 2 : kSmallBlocks) long_kernel(Rows a, Out o, int cluster, int shift) {
    __shared__ Shared sh;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / cluster;
    const Source<T, kMask> src(a, row);
    const int nv = src.vectors();
    const int each = ((nv + cluster - 1) / cluster + (1 << shift) - 1) >> shift << shift;
    const int v0 = min(nv, each * rank), v1 = min(nv, v0 + each);
    const float c = factor_of(a);
    if (kTop) {
        if (!kOnce)
            for (int i = threadIdx.x; i < kGroups; i += blockDim.x) sh.group[i] = 0;
        if (threadIdx.x == 0) sh.found = sh.chosen = 0;
        __syncthreads();
    }

    Action act{false, 0.0f};
    if (threadIdx.x == 0 && rank == 0) act = load_action<T>(a, o, row);
    uint4 q[kUnroll];
    Part p = empty_part();
    for (int base = v0 + warp * kTile; base < v1 || kOnce; base += warps * kTile) {
        if (base >= 2 && base + kTile <= min(v1, src.last())) {
#pragma unroll
            for (int u = 0; u < kUnroll; u++) q[u] = src.inner(base + u * 32 + lane);
        } else {
#pragma unroll
            for (int u = 0; u < kUnroll; u++) {
                const int v = base + u * 32 + lane;
                q[u] = v < v1 ? src.load(v) : no_vector<T>();
            }
        }
        float top[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) top[u] = most<T>(q[u]);
        const float here = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        if (kTop && !kOnce) {
            if (shift >= 7) {
                const uint32_t key = __reduce_max_sync(~0u, key_of(here));
                if (lane == 0) atomicMax(&sh.group[(base - v0) >> shift], key);
            } else {   // 5: a group is a warp's vectors of one u
#pragma unroll
                for (int u = 0; u < kUnroll; u++) {
                    const uint32_t key = __reduce_max_sync(~0u, key_of(top[u]));
                    if (lane == 0 && base + u * 32 < v1) sh.group[(base - v0) / 32 + u] = key;
                }
            }
        }
        const float m = max_nan(p.m, here);
        p = moved(p, m, reference(m, c));
        add_vectors<T, kUnroll, kMask>(q, c, p);
        if (kOnce) break;
    }
    const float mine = p.m;
    p = join_lanes(p);
    if (lane == 0) sh.part[warp] = p;
    if (kTop) {
        uint32_t key = sort_lanes(key_of(mine));
        sh.sorted[warp][lane] = key;
        int half = 1;
        while (half < warps) half *= 2;
        while (half /= 2) {
            __syncthreads();
            if (warp < half && warp + half < warps) {
                key = merge_lanes(key, sh.sorted[warp + half][31 - lane]);
                sh.sorted[warp][lane] = key;
            }
        }
    }
    __syncthreads();
    {   // each warp joins the warps' parts by its lanes
        p = lane < warps ? sh.part[lane] : empty_part();
        p = join_lanes(p);
    }

    if (kTop) {
        const int groups = (v1 - v0 + (1 << shift) - 1) >> shift;
        const uint32_t threshold = max(sh.sorted[0][o.top - 1], kNothing + 1);
        if (p.m != p.m) {
            search<T, kMask>(src, sh, v0, v1, shift, nullptr, groups, o.top);
        } else {
            if (!kOnce) {
                for (int g = threadIdx.x; g < groups; g += blockDim.x)
                    if (sh.group[g] >= threshold) sh.order[atomicAdd(&sh.chosen, 1)] = g;
                __syncthreads();
            }
            if (kOnce) {
#pragma unroll
                for (int u = 0; u < kUnroll; u++) gather(src, sh, q[u], v0 + warp * kTile + u * 32 + lane, threshold);
            } else {
                const int again = sh.chosen << shift;
                for (int i = threadIdx.x; i < again && *(volatile int*)&sh.found <= kFound; i += blockDim.x * kUnroll) {
                    int v[kUnroll];
#pragma unroll
                    for (int u = 0; u < kUnroll; u++) {
                        const int k = i + u * blockDim.x;
                        v[u] = k < again ? v0 + (sh.order[k >> shift] << shift) + (k & ((1 << shift) - 1)) : v1;
                        if (v[u] >= 2 && v[u] < min(v1, src.last())) q[u] = src.inner(v[u]);
                        else q[u] = v[u] < v1 ? src.load(v[u]) : no_vector<T>();
                    }
#pragma unroll
                    for (int u = 0; u < kUnroll; u++) gather(src, sh, q[u], v[u], threshold);
                }
            }
            __syncthreads();
            const int found = sh.found;
            if (found <= kFound) rank_entries(sh.entries, found, o.top, sh.list);
            else crowded<T, kMask, kOnce>(src, sh, v0, v1, shift, groups, o.top, threshold);
        }
        __syncthreads();
    }

    if (cluster > 1) {
        if (threadIdx.x == 0) sh.all = p;
        cluster_sync();
        if (rank == 0) {
            p = empty_part();
            if (lane < cluster)
                p = Part{remote_float(&sh.all.m, lane), remote_float(&sh.all.r, lane), remote_float(&sh.all.s, lane),
                         remote_float(&sh.all.t, lane)};
            p = join_lanes(p);
            if (kTop) {
                const int n = cluster * o.top;
                for (int i = threadIdx.x; i < n; i += blockDim.x) {
                    const uint64_t* at = &sh.list[i % o.top];
                    sh.entries[i] = (uint64_t)remote((const char*)at + 4, i / o.top) << 32 | remote(at, i / o.top);
                }
                if (threadIdx.x < o.top) sh.joined[threadIdx.x] = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < n; i += blockDim.x) {
                    const uint64_t e = sh.entries[i];
                    int rank = 0;
#pragma unroll 8
                    for (int j = 0; j < n; j++) rank += sh.entries[j] > e;
                    if (e && rank < o.top) sh.joined[rank] = e;
                }
                __syncthreads();
            }
        }
        cluster_sync();   // no block leaves while its shared memory is read
        if (rank) return;
    }
    const bool far = out_of_range(p, c);
    if (far) {
        const float2 st = far_sums(src, p.m, c, (int)threadIdx.x, (int)blockDim.x);
        if (lane == 0) sh.far[warp] = st;
        __syncthreads();
        p.s = p.t = 0.0f;
        for (int w = 0; w < warps; w++) p.s += sh.far[w].x, p.t += sh.far[w].y;
    }
    const Row r = far ? Row::about_maximum(p) : Row(p, c);
    if (threadIdx.x == 0) write_row(a, o, row, r, act);
    if (kTop)
        for (int k = threadIdx.x; k < o.top; k += blockDim.x)
            write_top(o, row, k, cluster > 1 ? sh.joined[k] : sh.list[k], r, a.scale);
}
static_assert(kMaxCluster * B3X_TRAIN_MAX_TOP <= kFound, "the blocks' alternatives are ranked at once");

template <class T, bool kMask, bool kTop>
int launch_long(const Rows& a, const Out& o, int nv, cudaStream_t s) {
    // A cluster a row while rows alone leave SMs idle and each block keeps 1,024 vectors: 8 rows of 131,072 bf16 with 20
    // alternatives 9.7 us, by single blocks 13.5; 8 rows of 32,768 8.1 us so, by two blocks each 10.2.
    int cluster = 1;
    while (cluster < kMaxCluster && a.rows * cluster * 2 <= 296 && nv / (cluster * 2) >= 1024) cluster *= 2;
    int each = (nv + cluster - 1) / cluster;
    // Rows for every SM several times over: small blocks, whose ends overlap (4,096 rows of 131,072 bf16 with 20
    // alternatives 254 us with 16 warps, 221 with 4; 2,048 masked rows of 50,001 120 us with 16, 75 with 2).  Fewer:
    // 16 warps (128 rows of 131,072 17 us, with 4 warps 24).
    const bool many = a.rows * cluster >= 592;
    const bool once = each <= (many ? 4 : kMaxWarps) * kTile;
    const int warps = once ? (each + kTile - 1) / kTile : !many ? kMaxWarps : each > 8192 ? 4 : 2;
    int shift = 0;
    if (!once) {
        shift = 5;   // 32 vectors a group, or 128 and more
        while ((each + (1 << shift) - 1) >> shift > kGroups) shift = shift == 5 ? 7 : shift + 1;
    }
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
    if (many)
        return (int)(once ? cudaLaunchKernelEx(&cfg, long_kernel<T, kMask, kTop, true, kSmallWarps>, a, o, cluster, shift)
                          : cudaLaunchKernelEx(&cfg, long_kernel<T, kMask, kTop, false, kSmallWarps>, a, o, cluster, shift));
    return (int)(once ? cudaLaunchKernelEx(&cfg, long_kernel<T, kMask, kTop, true, kMaxWarps>, a, o, cluster, shift)
                      : cudaLaunchKernelEx(&cfg, long_kernel<T, kMask, kTop, false, kMaxWarps>, a, o, cluster, shift));
}

template <class T, bool kMask, int L, bool kWalk>
int launch_lanes(const Rows& a, const Out& o, cudaStream_t s) {
    const long long per = kRowThreads / L;
    const unsigned grid = (unsigned)((a.rows + per - 1) / per);
    if (o.top) lanes_kernel<T, kMask, true, L, kWalk><<<grid, kRowThreads, 0, s>>>(a, o);
    else lanes_kernel<T, kMask, false, L, kWalk><<<grid, kRowThreads, 0, s>>>(a, o);
    return (int)cudaGetLastError();
}

// By the rows' vectors and number alone: a row's sums do not depend on what else is asked for.
template <class T, bool kMask>
int launch_rows(const Rows& a, const Out& o, cudaStream_t s) {
    // the most vectors that a row has
    const bool even = (uintptr_t)a.logits % 16 == 0 && a.row_stride * (long long)sizeof(T) % 16 == 0;
    const int nv = (int)(((long long)a.width + Vec<T>::n - 1) / Vec<T>::n) + (even ? 0 : 1);
    if (nv <= 8) return launch_lanes<T, kMask, 2, false>(a, o, s);
    if (nv <= 16) return launch_lanes<T, kMask, 4, false>(a, o, s);
    if (nv <= 32) return launch_lanes<T, kMask, 8, false>(a, o, s);
    if (nv <= 64) return launch_lanes<T, kMask, 16, false>(a, o, s);
    if (nv <= 128) return launch_lanes<T, kMask, 32, false>(a, o, s);
    // a warp a row up to some thousand logits, where rows fill the SMs (8,192 rows of 16,384 bf16 with 20 alternatives
    // 92 us, by blocks 101; 2,048 rows of 50,001 f16 103, by blocks 53)
    if (nv <= 2048 && a.rows >= 8 * 148) return launch_lanes<T, kMask, 32, true>(a, o, s);
    return o.top ? launch_long<T, kMask, true>(a, o, nv, s) : launch_long<T, kMask, false>(a, o, nv, s);
}

template <class T>
int launch(const Rows& a, const Out& o, cudaStream_t s) {
    if (a.width <= kShort) {
        short_kernel<T><<<(unsigned)((a.rows + kShortThreads - 1) / kShortThreads), kShortThreads, 0, s>>>(a, o);
        return (int)cudaGetLastError();
    }
    return a.mask ? launch_rows<T, true>(a, o, s) : launch_rows<T, false>(a, o, s);
}



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
