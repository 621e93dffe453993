// b3x_train_rows.cuh -- rows of logits as the kernels read them: 16 bytes at a
// time on the boundaries of memory, masked places as -infinity (b3x_train.h).
#pragma once
#include <cmath>

#include "b3x_train_common.cuh"

namespace b3t {

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

// 16 bytes of consecutive logits.  A row is cut on the 16-byte boundaries of
// memory, wherever it starts: vector v holds the elements from v N - head on.
template <class T> struct Vec { static constexpr int n = 16 / sizeof(T); };

// kAgain: will be read again soon, so it stays in L1.
template <bool kAgain>
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 q;
    if (kAgain)
        asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
    else
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

// A row's vectors.  Whole 16 bytes are read wherever they lie within the tensor,
// so that the ends of a row that starts off a boundary cost no loads of their
// own: what belongs to its neighbours, or to the space between rows, is replaced.
template <class T, bool kMask, bool kAgain = false>
struct Source {
    static constexpr int N = Vec<T>::n;
    const T* row;
    const unsigned char* mask;
    const T *begin, *end;                         // the tensor's
    const unsigned char *mask_begin, *mask_end;   // the mask's
    int width, head;

    __device__ __forceinline__ Source(const Rows& a, long long r) {
        begin = (const T*)a.logits;
        end = begin + (a.rows - 1) * a.row_stride + a.width;
        row = begin + r * a.row_stride;
        mask_begin = kMask ? a.mask : nullptr;
        mask_end = kMask ? a.mask + (a.rows - 1) * a.mask_stride + a.width : nullptr;
        mask = kMask ? a.mask + r * a.mask_stride : nullptr;
        width = a.width;
        head = (int)((uintptr_t)row % 16 / sizeof(T));
    }
    __device__ __forceinline__ int vectors() const { return (head + width + N - 1) / N; }

    // Vectors [2, last) and two words beside them are inside the row.
    __device__ __forceinline__ int last() const { return (head + width) / N - 1; }
    // A vector among those.
    __device__ __forceinline__ uint4 inner(int v) const {
        const int j = v * N - head;
        uint4 q = load16<kAgain>(row + j);
        if (kMask) keep(q, mask + j);
        return q;
    }

    // Vector v, -infinity where it is outside the row or masked.
    __device__ __forceinline__ uint4 load(int v) const {
        const int j = v * N - head;
        const bool ends = j < 0 || j + N > width;
        uint4 q;
        if (!ends || (row + j >= begin && row + j + N <= end)) {
            q = load16<kAgain>(row + j);
        } else {
            uint32_t* w = &q.x;
            w[0] = w[1] = w[2] = w[3] = 0;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (j + i < 0 || j + i >= width) continue;
                if (sizeof(T) == 4) w[i % 4] = reinterpret_cast<const uint32_t*>(row)[j + i];
                else w[i / 2 % 4] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[j + i] << i % 2 * 16;
            }
        }
        if (kMask) apply(q, j);
        if (ends) {
            uint32_t* w = &q.x;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = j + i * (N / 4);
                if (sizeof(T) == 4) {
                    if (k < 0 || k >= width) w[i] = minus_infinity<T>();
                } else {
                    if (k < 0 || k >= width) w[i] = (w[i] & 0xFFFF0000u) | (minus_infinity<T>() & 0xFFFFu);
                    if (k + 1 < 0 || k + 1 >= width) w[i] = (w[i] & 0xFFFFu) | (minus_infinity<T>() & 0xFFFF0000u);
                }
            }
        }
        return q;
    }

    // Mask bytes j on, where the words around them may lie outside the mask.
    __device__ __forceinline__ void apply(uint4& q, int j) const {
        const unsigned char* p = mask + j;
        const int off = (int)((uintptr_t)p & 3);
        if (p - off >= mask_begin && p - off + N + 4 <= mask_end) return keep(q, p);
        uint32_t b[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < N; i++)
            if (j + i >= 0 && j + i < width) b[i / 4] |= (uint32_t)p[i] << i % 4 * 8;
        keep(q, b);
    }

    // The N mask bytes at p, from the whole words around them.
    static __device__ __forceinline__ void keep(uint4& q, const unsigned char* p) {
        const int off = (int)((uintptr_t)p & 3);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(p - off);
        const uint32_t w0 = __ldg(w), w1 = N == 8 || off ? __ldg(w + 1) : 0u, w2 = N == 8 && off ? __ldg(w + 2) : 0u;
        uint32_t b[2] = {__funnelshift_r(w0, w1, off * 8), __funnelshift_r(w1, w2, off * 8)};
        keep(q, b);
    }

    static __device__ __forceinline__ void keep(uint4& q, uint32_t (&b)[2]) {
        uint32_t* w = &q.x;
        b[0] = nonzero_bytes(b[0]);
        if (N == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = b[0] >> i * 8 & 0x80u ? w[i] : minus_infinity<T>();
        } else {
            b[1] = nonzero_bytes(b[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) {   // a byte's sign bit becomes 16 bits of ones
                uint32_t ones;
                asm("prmt.b32 %0, %1, 0, %2;" : "=r"(ones) : "r"(b[i / 2]), "r"(i % 2 ? 0xBBAA : 0x9988));
                w[i] = (w[i] & ones) | (minus_infinity<T>() & ~ones);
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

template <class T> __device__ __forceinline__ uint4 no_vector() {
    return make_uint4(minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>(), minus_infinity<T>());
}

inline bool rows_ok(const void* logits, int type, long long rows, long long width, long long row_stride,
             const unsigned char* mask, long long mask_stride, const void* actions, int action_bytes, float scale) {
    if (type < B3X_F32 || type > B3X_F16 || rows < 0 || rows > 0x7fffffff || !(scale > 0.0f) || !std::isfinite(scale))
        return false;
    if (rows == 0) return true;
    if (width < 1 || width > (1ll << 30) || row_stride < 0 || mask_stride < 0 || !logits) return false;
    if ((uintptr_t)logits % (type == B3X_F32 ? 4 : 2)) return false;
    if (actions && action_bytes != 4 && action_bytes != 8) return false;
    return !actions || (uintptr_t)actions % action_bytes == 0;
}

inline bool aligned4(const void* p) { return (uintptr_t)p % 4 == 0; }

}  // namespace b3t
