// ml_common.cuh — element types, vector loads and stores, and activations
// shared by the decoder operators (RMS norm, matrix product with epilogue).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "qc_common.cuh"

namespace qc {
namespace ml {

template <int T>
struct ElemOf;
template <>
struct ElemOf<QC_F32> { using type = float; };
template <>
struct ElemOf<QC_BF16> { using type = __nv_bfloat16; };
template <>
struct ElemOf<QC_F16> { using type = __half; };

__host__ __device__ __forceinline__ int elem_size(int t) {
    return t == QC_F32 ? 4 : t == QC_E4M3 ? 1 : 2;
}

template <int BYTES>
struct alignas(BYTES) Bits {
    unsigned char b[BYTES];
};

// V values of type T as they lie in memory: what a load keeps in registers
// until the values are needed (a 16-bit value costs half a register).
template <int T, int V>
struct Raw {
    using E = typename ElemOf<T>::type;
    static constexpr int kBytes = V * (int)sizeof(E);
    union {
        Bits<kBytes> bits;
        uint32_t w[kBytes >= 4 ? kBytes / 4 : 1];
    };

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (kBytes >= 4 ? kBytes / 4 : 1); ++i) w[i] = 0;
    }
    // p must be aligned to kBytes (up to 32: one 256-bit access)
    __device__ __forceinline__ void load(const void *base, long long idx) {
        const E *p = static_cast<const E *>(base) + idx;
        if constexpr (kBytes == 16) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (kBytes == 32) {
            asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                : "l"(p));
        } else if constexpr (kBytes == 8) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            w[0] = *reinterpret_cast<const unsigned short *>(p);
        }
    }
    // Values lo <= i < hi one by one, from any address of the type; 0 elsewhere.
    __device__ __forceinline__ void load_some(const void *base, long long idx, int lo, int hi) {
        const E *p = static_cast<const E *>(base) + idx;
        zero();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= lo && i < hi) {
                if constexpr (T == QC_F32)
                    w[i] = reinterpret_cast<const uint32_t *>(p)[i];
                else
                    w[i / 2] |= (uint32_t) reinterpret_cast<const unsigned short *>(p)[i] << (16 * (i & 1));
            }
    }
    // Zeroes the values outside lo <= i < hi.
    __device__ __forceinline__ void keep(int lo, int hi) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < lo || i >= hi) {
                if constexpr (T == QC_F32) w[i] = 0;
                else w[i / 2] &= i & 1 ? 0xffffu : 0xffff0000u;
            }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (T == QC_F32) {
            return __uint_as_float(w[i]);
        } else {
            const unsigned short h = (unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
            if constexpr (T == QC_BF16)
                return __uint_as_float((uint32_t)h << 16);
            else
                return __half2float(__ushort_as_half(h));
        }
    }
};

// Two values in one 64-bit register: one instruction per operation for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ Pair pair(float a) { return pair(a, a); }
__device__ __forceinline__ void split(Pair p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// four values as e4m3, rounded to nearest even, the largest finite value
// beyond the range (NaN stays NaN)
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// One value of runtime type t.
__device__ __forceinline__ float load_any(const void *base, long long i, int t) {
    if (t == QC_F32) return static_cast<const float *>(base)[i];
    if (t == QC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(base)[i]);
    return __half2float(static_cast<const __half *>(base)[i]);
}
__device__ __forceinline__ void store_any(void *base, long long i, int t, float v) {
    if (t == QC_F32)
        static_cast<float *>(base)[i] = v;
    else if (t == QC_BF16)
        static_cast<__nv_bfloat16 *>(base)[i] = __float2bfloat16_rn(v);
    else if (t == QC_F16)
        static_cast<__half *>(base)[i] = __float2half_rn(v);
    else
        static_cast<unsigned char *>(base)[i] = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// V values of runtime type t (uniform over the launch) to a V-aligned place.
template <int V>
__device__ __forceinline__ void store_vec(void *base, long long i, int t, const float (&v)[V]) {
    if constexpr (V == 1) {
        store_any(base, i, t, v[0]);
    } else {
        static_assert(V == 4 || V == 8, "4 or 8 values");
        if (t == QC_F32) {
            float *p = static_cast<float *>(base) + i;
            if constexpr (V == 8)
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]),
                             "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                             : "memory");
            else
                *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else if (t == QC_E4M3) {
            uint32_t w[V / 4];
#pragma unroll
            for (int q = 0; q < V / 4; ++q)
                w[q] = pack_e4m3x4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            unsigned char *p = static_cast<unsigned char *>(base) + i;
            if constexpr (V == 8)
                *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t *>(p) = w[0];
        } else {
            uint32_t w[V / 2];
#pragma unroll
            for (int q = 0; q < V / 2; ++q)
                w[q] = t == QC_BF16 ? pack_bf16(v[2 * q], v[2 * q + 1]) : pack_f16(v[2 * q], v[2 * q + 1]);
            unsigned short *p = static_cast<unsigned short *>(base) + i;
            if constexpr (V == 8)
                *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            else
                *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        }
    }
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ── column sums ───────────────────────────────────────────────────────────
// out[c] = sum over p of partial[p*n + c] in a fixed order, rounded once to
// out_type; two launches' worth of partial sums (weight and bias gradients).
int launch_colsum_reduce(const float *partial, int parts, int n, void *out, int out_type, cudaStream_t stream);

bool aligned_to(const void *p, long long bytes);

// The norms' fault word (the products' is ml_fault_word's own).
int norm_fault_word(unsigned int *word, int clear);

}  // namespace ml
}  // namespace qc
