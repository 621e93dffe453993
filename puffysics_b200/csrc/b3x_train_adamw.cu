// b3x_train_adamw.cu -- the global norm of a list of gradients and one AdamW
// step over a list of tensors (b3x_train.h).
#include <cmath>

#include "b3x_train_common.cuh"

using namespace b3t;

namespace {

constexpr int kThreads = 256;
constexpr int kTurn = kThreads * 8;     // elements a block takes at a time: a scale's 256 for each warp
constexpr int kNormBlocks = 592;        // partial sums of the norm
constexpr int kFew = 16, kMany = 256;   // tensors of one launch: their table travels in the kernel's parameters
static_assert(B3X_TRAIN_BLOCK == 256, "a warp's 8 elements a lane share a scale");

struct Tensor {
    void* p;
    const void* g;
    void *m, *v;
    float* scales;
    __nv_bfloat16* copy;
    long long n;
    float keep;          // 1 - lr weight_decay
    unsigned key;        // the tensor's part of the rounding hash
    int even;            // every array starts at a multiple of 4 elements
};

template <int N>
struct List {
    int count, turns;        // turns of a chunk
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

// Four consecutive elements.
template <class T> __device__ __forceinline__ void load4(float (&x)[4], const T* p);
template <> __device__ __forceinline__ void load4(float (&x)[4], const float* p) {
    const float4 w = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
}
template <> __device__ __forceinline__ void load4(float (&x)[4], const __nv_bfloat16* p) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
    x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xFFFF0000u);
    x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void load4(float (&x)[4], const __half* p) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b)));
}

// Two e4m3 codes' values.
__device__ __forceinline__ float2 decode2(unsigned codes) {
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)codes));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The e4m3 code of |y| <= 448 in the upper byte.  Scaled by 2^-120 the format's
// exponents are float's, subnormals included, so the code is the word from bit
// 20 on; what is added to the 20 bits below it rounds: random bits up or down in
// proportion (16 of them, and a half of the last), a half to nearest.  448 and
// its next neighbours, which a product may round to, never carry beyond the
// largest code.
template <bool kRandom>
__device__ __forceinline__ uint32_t encode(float y, uint32_t bits16_at4) {
    const uint32_t w = __float_as_uint(fabsf(y) * 0x1p-120f);
    return (w + (kRandom ? (bits16_at4 & 0xFFFF0u) | 8u : 0x7FFFFu + ((w >> 20) & 1u))) << 4;
}

// The upper bytes of four words.
__device__ __forceinline__ uint32_t upper_bytes(const uint32_t (&w)[4]) {
    return __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
}

// A sum of products that rounds by itself: a two-wide addition would be fused with one of them.
__device__ __forceinline__ uint64_t sum2(uint64_t a, uint64_t b) {
    const float2 x = unpack2(a), y = unpack2(b);
    return pack2(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}

// The largest of three numbers' magnitudes, NaN above all.
__device__ __forceinline__ float most3(float a, float b, float c) {
    float y;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ float reciprocal(float x) {   // 1 ulp
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The least of three numbers, NaN below all.
__device__ __forceinline__ float least3(float a, float b, float c) {
    float y;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// The largest of a warp's numbers that are not negative; NaN is the largest.
__device__ __forceinline__ float warp_most(float x) {
    return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(x) & 0x7FFFFFFFu));
}

// A warp takes the 256 elements of one scale at a time, two runs of four a lane,
// so that every load and store is a whole line however wide its type.  The
// moments' operations round one by one: their codes are those of the plain
// formula, bit for bit.
//
// 168 M parameters.  In 32 bits throughout 704 us, 6.8 TB/s, a little over the
// copy rate: bound by memory (bf16 parameters and gradients 558 us, 6.8 TB/s).
// With 8-bit moments, bf16 parameters and gradients and stochastic rounding 451
// us, 59% of the copy rate: bound by issued instructions, 79 an element (issue
// slots 77% busy, the integer pipe 63%), of which the two hashes are 19 and the
// codes 12.  Elements one by one, where any of a tensor's arrays is off a
// boundary of four: 1,083 us for 731 in 32 bits, 685 for 463 with 8-bit moments
// (176 M parameters).
template <class P, class G, bool kF8, bool kRandom, bool kWhole>
__device__ __forceinline__ void update(const Tensor& t, const Hyper& h, const float gs, const long long base, const int lane) {
    const long long n = t.n;
    P* const pp = (P*)t.p;
    const G* const pg = (const G*)t.g;
    float p[2][4], g[2][4], m[2][4], v[2][4];
    uint32_t cm[2], cv[2];
    float sm = 0.0f, sr = 0.0f;
    if (kF8) {
        const float2 s = *reinterpret_cast<const float2*>(t.scales + base / 256 * 2);
        sm = s.x, sr = s.y;
    }
    if (kWhole) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long i = base + k * 128 + lane * 4;
            load4(g[k], pg + i);
            load4(p[k], pp + i);
            if (kF8) {
                cm[k] = __ldcs(reinterpret_cast<const uint32_t*>((const unsigned char*)t.m + i));
                cv[k] = __ldcs(reinterpret_cast<const uint32_t*>((const unsigned char*)t.v + i));
            } else {
                load4(m[k], (const float*)t.m + i);
                load4(v[k], (const float*)t.v + i);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            cm[k] = cv[k] = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const long long i = base + k * 128 + lane * 4 + j;
                const bool in = i < n;
                g[k][j] = in ? to_float(pg[i]) : 0.0f;
                p[k][j] = in ? to_float(pp[i]) : 0.0f;
                if (kF8) {
                    cm[k] |= in ? (uint32_t)((const unsigned char*)t.m)[i] << j * 8 : 0u;
                    cv[k] |= in ? (uint32_t)((const unsigned char*)t.v)[i] << j * 8 : 0u;
                } else {
                    m[k][j] = in ? ((const float*)t.m)[i] : 0.0f;
                    v[k][j] = in ? ((const float*)t.v)[i] : 0.0f;
                }
            }
        }
    }
    float most_m = 0.0f, most_r = 0.0f, most_p = 0.0f;
    const uint64_t gs2 = pack2(gs, gs), sm2 = pack2(sm, sm), sr2 = pack2(sr, sr), b1 = pack2(h.b1, h.b1), c1 = pack2(h.c1, h.c1),
                   b2 = pack2(h.b2, h.b2), c2 = pack2(h.c2, h.c2), root = pack2(h.root, h.root), eps = pack2(h.eps, h.eps),
                   keep = pack2(t.keep, t.keep), rate = pack2(-h.rate, -h.rate);
    float least_v = kInf, most_v = 0.0f;
    uint64_t m2[4], v2[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int k = q / 2, j = q % 2 * 2;
        if (kF8) {
            const float2 a = decode2(cm[k] >> j * 8), b = decode2(cv[k] >> j * 8);
            m2[q] = mul2(pack2(a.x, a.y), sm2);
            const uint64_t r = mul2(pack2(b.x, b.y), sr2);
            v2[q] = mul2(r, r);
        } else {
            m2[q] = pack2(m[k][j], m[k][j + 1]);
            v2[q] = pack2(v[k][j], v[k][j + 1]);
        }
        const uint64_t x = mul2(pack2(g[k][j], g[k][j + 1]), gs2);
        m2[q] = sum2(mul2(m2[q], b1), mul2(x, c1));
        v2[q] = sum2(mul2(v2[q], b2), mul2(mul2(x, x), c2));
        const float2 vv = unpack2(v2[q]);
        least_v = least3(least_v, vv.x, vv.y), most_v = most3(most_v, vv.x, vv.y);
    }
    const bool usual = least_v >= 0x1p-96f && most_v <= 0x1p100f;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int k = q / 2, j = q % 2 * 2;
        const float2 vv = unpack2(v2[q]), nm = unpack2(m2[q]);
        float2 r = unpack2(sqrt2(v2[q]));
        if (!usual) r = make_float2(sqrtf(vv.x), sqrtf(vv.y));
        const float2 d = unpack2(fma2(pack2(r.x, r.y), root, eps));
        const uint64_t step = mul2(mul2(m2[q], pack2(reciprocal(d.x), reciprocal(d.y))), rate);
        const float2 np = unpack2(fma2(pack2(p[k][j], p[k][j + 1]), keep, step));
        p[k][j] = np.x, p[k][j + 1] = np.y;
        m[k][j] = nm.x, m[k][j + 1] = nm.y;
        if (kF8) {
            most_m = most3(most_m, nm.x, nm.y), most_r = most3(most_r, r.x, r.y);
            v[k][j] = r.x, v[k][j + 1] = r.y;
        } else {
            v[k][j] = vv.x, v[k][j + 1] = vv.y;
        }
        if (kRandom && sizeof(P) == 2) most_p = most3(most_p, np.x, np.y);
    }
    if (!kF8) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long i = base + k * 128 + lane * 4;
            if (kWhole) {
                store4((float*)t.m + i, m[k]);
                store4((float*)t.v + i, v[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i + j < n) ((float*)t.m)[i + j] = m[k][j], ((float*)t.v)[i + j] = v[k][j];
            }
        }
    }
    if (t.copy) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long i = base + k * 128 + lane * 4;
            if (kWhole) {
                store4(t.copy + i, p[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i + j < n) t.copy[i + j] = __float2bfloat16_rn(p[k][j]);
            }
        }
    }
    uint32_t bits[2][4];
    if (kRandom) {
        const uint32_t at = (uint32_t)(base + lane * 4) * 0x9E3779B1u + (uint32_t)(base >> 32) * 0x6A09E667u + t.key;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) bits[k][j] = mix(at + (k * 128 + j) * 0x9E3779B1u);
    }
    if (kRandom && sizeof(P) == 2) {
        uint32_t low[2][4];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) low[k][j] = mix(bits[k][j] + 0x9E3779B1u) & 0xFFFFu;
        if (most_p != most_p) {   // NaN stays what it is
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (p[k][j] != p[k][j]) low[k][j] = 0;
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long i = base + k * 128 + lane * 4;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = __float_as_uint(p[k][j]) + low[k][j];
            const uint2 q = make_uint2(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
            if (kWhole) {
                __stcs(reinterpret_cast<uint2*>(pp + i), q);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i + j < n) reinterpret_cast<uint16_t*>(pp)[i + j] = (uint16_t)(w[j] >> 16);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long i = base + k * 128 + lane * 4;
            if (kWhole) {
                store4(pp + i, p[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i + j < n) pp[i + j] = from_float<P>(p[k][j]);
            }
        }
    }
    if (!kF8) return;
    most_m = warp_most(most_m), most_r = warp_most(most_r);
    // a division for each quarter of the lanes: the scales, and what makes codes of the moments
    const float most = lane < 16 ? most_m : most_r;
    const float part = most < 0x1p-100f ? 0.0f : lane & 8 ? 448.0f / most : most / 448.0f;
    if ((lane & 15) == 0) t.scales[base / 256 * 2 + lane / 16] = part;
    const float im = __shfl_sync(~0u, part, 8), ir = __shfl_sync(~0u, part, 24);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint32_t wm[4], wv[4], sign[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            wm[j] = encode<kRandom>(m[k][j] * im, bits[k][j] << 4);
            wv[j] = encode<kRandom>(v[k][j] * ir, bits[k][j] >> 12);
            sign[j] = __float_as_uint(m[k][j]);
        }
        cm[k] = upper_bytes(wm) | (upper_bytes(sign) & 0x80808080u);
        cv[k] = upper_bytes(wv);
        // a moment above zero never becomes zero: it would divide by eps alone
        if (((cv[k] + 0x7F7F7F7Fu) & 0x80808080u) != 0x80808080u && ir != 0.0f) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (v[k][j] > 0.0f && !(cv[k] >> j * 8 & 0xFFu)) cv[k] |= 1u << j * 8;
        }
        const long long i = base + k * 128 + lane * 4;
        if (kWhole) {
            __stcs(reinterpret_cast<uint32_t*>((unsigned char*)t.m + i), cm[k]);
            __stcs(reinterpret_cast<uint32_t*>((unsigned char*)t.v + i), cv[k]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < n) {
                    ((unsigned char*)t.m)[i + j] = (unsigned char)(cm[k] >> j * 8);
                    ((unsigned char*)t.v)[i + j] = (unsigned char)(cv[k] >> j * 8);
                }
        }
    }
}

// kWhole: all 256 elements, every array at a multiple of 4 of them.
template <class P, class G, bool kF8, bool kRandom, int N>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ List<N> list, const Hyper h) {
    const float gs = h.grad_scale ? *h.grad_scale : 1.0f;
    if (!(fabsf(gs) < kInf)) return;
    const int which = find(list, blockIdx.x);
    const Tensor& t = list.t[which];
    const int lane = threadIdx.x % 32;
    long long base = ((long long)(blockIdx.x - list.first[which]) * list.turns * (kTurn / 256) + threadIdx.x / 32) * 256;
    for (int turn = 0; turn < list.turns && base < t.n; turn++, base += kTurn) {
        if (t.even && base + 256 <= t.n) update<P, G, kF8, kRandom, true>(t, h, gs, base, lane);
        else update<P, G, kF8, kRandom, false>(t, h, gs, base, lane);
    }
}

// ---- norm -------------------------------------------------------------------------------
__device__ __forceinline__ double square(float x) { return (double)x * (double)x; }

// A block's sum over its chunks, on its first thread.
template <class G, int N>
__device__ __forceinline__ double sum_squares(const List<N>& list, double* buf) {
    double s = 0.0;
    const unsigned chunks = list.first[list.count];
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int k = find(list, c);
        const Tensor& t = list.t[k];
        const G* g = (const G*)t.g;
        const long long begin = (long long)(c - list.first[k]) * list.turns * kTurn;
        for (int turn = 0; turn < list.turns; turn++) {
            const long long base = begin + turn * kTurn;
            if (base >= t.n) break;
            if (t.even && base + kTurn <= t.n) {
                float x[2][4];
#pragma unroll
                for (int u = 0; u < 2; u++) load4(x[u], g + base + (u * kThreads + threadIdx.x) * 4);
#pragma unroll
                for (int u = 0; u < 2; u++) s += (square(x[u][0]) + square(x[u][1])) + (square(x[u][2]) + square(x[u][3]));
            } else {
                for (int u = 0; u < 8; u++) {
                    const long long i = base + u * kThreads + threadIdx.x;
                    if (i < t.n) s += square(to_float(g[i]));
                }
            }
        }
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < kThreads / 32; i++) s += buf[i];
    return s;
}

__device__ __forceinline__ void write_norm(double s, float max_norm, float* out) {
    const float norm = (float)sqrt(s);
    out[0] = norm;
    out[1] = fabsf(norm) < kInf ? fminf(1.0f, max_norm / (norm + 1e-6f)) : norm - norm;
}

template <class G, int N>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ List<N> list, double* sums, int more) {
    __shared__ double buf[kThreads / 32];
    const double s = sum_squares<G>(list, buf);
    if (threadIdx.x == 0) sums[blockIdx.x] = more ? sums[blockIdx.x] + s : s;
}

__global__ void __launch_bounds__(kThreads) norm_end_kernel(const double* sums, float max_norm, float* out) {
    __shared__ double buf[kThreads / 32];
    double s = 0.0;
    for (int i = threadIdx.x; i < kNormBlocks; i += kThreads) s += sums[i];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / 32; i++) s += buf[i];
        write_norm(s, max_norm, out);
    }
}

// Few elements: one cluster, whose first block joins the sums (the hover policy's
// clip and step 6.1 us, with the two launches 6.8).
constexpr int kNormCluster = 8;
constexpr long long kNormSmall = 1 << 18;   // elements

template <class G>
__global__ void __launch_bounds__(kThreads) norm_small_kernel(const __grid_constant__ List<kFew> list, float max_norm, float* out) {
    __shared__ double buf[kThreads / 32], sum;
    const double s = sum_squares<G>(list, buf);
    if (threadIdx.x == 0) sum = s;
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        double all = s;
        for (int r = 1; r < kNormCluster; r++) {
            unsigned at;
            double x;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(&sum)), "r"(r));
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(at) : "memory");
            all += x;
        }
        write_norm(all, max_norm, out);
    }
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}

int bytes_of(int type) { return type == B3X_F32 ? 4 : type == B3X_E4M3 || type == B3X_U8 ? 1 : 2; }

bool at(const void* p, int bytes) { return p && (uintptr_t)p % bytes == 0; }

// Fills lists of at most N tensors and hands each to `go`; tensors without elements are left out.
template <int N, class Fill, class Go>
int each_list(int count, const long long* sizes, int turns, Fill fill, Go go) {
    List<N> list;
    list.turns = turns;
    const long long chunk = (long long)turns * kTurn;
    int k = 0;
    bool more = false;
    while (k < count) {
        list.count = 0;
        list.first[0] = 0;
        for (; k < count && list.count < N; k++) {
            if (sizes[k] == 0) continue;
            const long long chunks = (sizes[k] + chunk - 1) / chunk;
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

// Turns of a chunk: one while there are few, so that all SMs have some; then as
// many as spread a block's start over its work (168 M parameters, with a clip and
// 32-bit moments: 859 us with one turn, 831 with 4, 845 with 8; with 8-bit
// moments 541, 460, 449).  Just above the edge 8 turns leave a tail of blocks that
// fill the SMs in part: 10 M parameters with 8-bit moments 38.2 us, with one turn
// 34.1; 12 M 42.7 and 39.7; 16 M 51.2 and 52.5; 40 M 114 and 124.
int turns_for(int count, const long long* sizes, int most) {
    long long all = 0;
    for (int k = 0; k < count; k++) all += sizes[k];
    return all / kTurn >= 148 * 32 ? most : 1;
}

// Whether p is at a multiple of 4 elements of `bytes` (or absent).
int even(const void* p, int bytes) { return (uintptr_t)p % (4 * bytes) == 0; }

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
    const int bytes = bytes_of(grad_type);
    int used = 0;
    long long all = 0;
    for (int k = 0; k < count; k++) used += sizes[k] > 0, all += sizes[k];
    auto fill = [&](int k) {
        return Tensor{nullptr, grads[k], nullptr, nullptr, nullptr, nullptr, sizes[k], 0.0f, 0, even(grads[k], bytes)};
    };
    if (used == 0) {
        const cudaError_t z = cudaMemsetAsync(sums, 0, kNormBlocks * sizeof(double), s);
        if (z != cudaSuccess) return (int)z;
    } else if (used <= kFew && all <= kNormSmall) {
        cudaError_t e = cudaSuccess;
        const int rc = each_list<kFew>(count, sizes, 1, fill, [&](const List<kFew>& list, bool) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(kNormCluster);
            cfg.blockDim = dim3(kThreads);
            cfg.stream = s;
            cudaLaunchAttribute attribute[1];
            attribute[0].id = cudaLaunchAttributeClusterDimension;
            attribute[0].val.clusterDim.x = kNormCluster;
            attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
            cfg.attrs = attribute;
            cfg.numAttrs = 1;
            const float limit = (float)max_norm;
            if (grad_type == B3X_F32) e = cudaLaunchKernelEx(&cfg, norm_small_kernel<float>, list, limit, out);
            if (grad_type == B3X_BF16) e = cudaLaunchKernelEx(&cfg, norm_small_kernel<__nv_bfloat16>, list, limit, out);
            if (grad_type == B3X_F16) e = cudaLaunchKernelEx(&cfg, norm_small_kernel<__half>, list, limit, out);
        });
        return rc ? rc : (int)e;
    }
    const int e = each_list<kMany>(count, sizes, turns_for(count, sizes, 4), fill, [&](const List<kMany>& list, bool more) {
        if (grad_type == B3X_F32) norm_kernel<float><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
        if (grad_type == B3X_BF16) norm_kernel<__nv_bfloat16><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
        if (grad_type == B3X_F16) norm_kernel<__half><<<kNormBlocks, kThreads, 0, s>>>(list, sums, more);
    });
    if (e) return e;
    norm_end_kernel<<<1, kThreads, 0, s>>>(sums, (float)max_norm, out);
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
    // The reciprocal of sqrt(v) root + eps takes numbers under the normal floats for 0: where eps is near those, both
    // terms and the rate are 2^24 times as large.
    const float up = (float)eps > 0.0f && (float)eps < 0x1p-100f ? 0x1p24f : 1.0f;
    const Hyper h{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2),
                  (float)(lr / (1.0 - std::pow(beta1, t))) * up, (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, t))) * up,
                  (float)eps * up, grad_scale};
    const cudaStream_t s = (cudaStream_t)stream;
    auto fill = [&](int k) {
        const double wd = decays ? (double)decays[k] : weight_decay;
        const unsigned key = mix(seed + (unsigned)k * 0x9E3779B1u + (unsigned)(unsigned long long)step * 0x6A09E667u);
        return Tensor{params[k], grads[k], exp_avg[k], exp_avg_sq[k], f8 ? scales[k] : nullptr,
                      copies ? (__nv_bfloat16*)copies[k] : nullptr, sizes[k], (float)(1.0 - lr * wd), key,
                      even(params[k], bytes_of(param_type)) && even(grads[k], bytes_of(grad_type)) &&
                          even(exp_avg[k], bytes_of(state_type)) && even(exp_avg_sq[k], bytes_of(state_type)) &&
                          even(copies ? copies[k] : nullptr, 2)};
    };
    auto go = [&](const auto& list, bool) {
        const unsigned grid = list.first[list.count];
#define B3T_GO(P, G)                                                                                        \
        (f8 ? stochastic ? adamw_kernel<P, G, true, true><<<grid, kThreads, 0, s>>>(list, h)                \
                         : adamw_kernel<P, G, true, false><<<grid, kThreads, 0, s>>>(list, h)               \
            : stochastic && sizeof(P) == 2 ? adamw_kernel<P, G, false, sizeof(P) == 2><<<grid, kThreads, 0, s>>>(list, h) \
                         : adamw_kernel<P, G, false, false><<<grid, kThreads, 0, s>>>(list, h))
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
    int used = 0;
    for (int k = 0; k < count; k++) used += sizes[k] > 0;
    const int turns = turns_for(count, sizes, f8 ? 8 : 4);
    return used <= kFew ? each_list<kFew>(count, sizes, turns, fill, go) : each_list<kMany>(count, sizes, turns, fill, go);
}
