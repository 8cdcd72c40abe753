// bfa_rows.hpp -- what the row operators (bfa_norm.hip, bfa_loss.hip, bfa_sample.hip) share: rows [B, T, C] of float32 /
// float16 / bfloat16 with a batch and a row stride, T_len[b] of them held, and reductions over 4, 16 or 64 lanes or a workgroup.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/bfa.h"

namespace bfa {

// n / d for 32-bit n by a multiplication (round-up method of Granlund and Montgomery, 1994)
struct FastDiv {
    uint32_t d, m, s1, s2;
    explicit FastDiv(uint32_t d_ = 1) : d(d_)
    {
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < d) ++l;
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
        s1 = l < 1 ? l : 1;
        s2 = l < 1 ? 0 : l - 1;
    }
#ifdef __HIPCC__
    __device__ __forceinline__ uint32_t div(uint32_t n) const
    {
        const uint32_t t = __umulhi(m, n);
        return (t + ((n - t) >> s1)) >> s2;
    }
#endif
};

// the rows of one call: row r = (b, t) = (r / T, r % T); B * T < 2^31 (the C entry checks)
struct RowShape {
    uint32_t rows, T;
    int C;
    const int32_t *len; // T_len or null
    FastDiv byT;
    RowShape(int B, int T_, int C_, const int32_t *len_) : rows((uint32_t)((int64_t)B * T_)), T((uint32_t)T_), C(C_), len(len_), byT((uint32_t)T_) {}
#ifdef __HIPCC__
    __device__ __forceinline__ void split(uint32_t r, uint32_t &b, uint32_t &t) const { b = byT.div(r); t = r - b * T; }
    __device__ __forceinline__ bool held(uint32_t b, uint32_t t) const { return !len || (int)t < len[b]; }
#endif
};
struct RowPtr {
    const void *p;
    int64_t sB, sT; // elements
};

#ifdef __HIPCC__
template <typename T> __device__ __forceinline__ const T *row_in(const RowPtr &x, uint32_t b, uint32_t t)
{
    return (const T *)x.p + (int64_t)b * x.sB + (int64_t)t * x.sT;
}
template <typename T> __device__ __forceinline__ T *row_out(const RowPtr &x, uint32_t b, uint32_t t)
{
    return (T *)const_cast<void *>(x.p) + (int64_t)b * x.sB + (int64_t)t * x.sT;
}
// N elements from an address that is aligned to one element only (the hardware takes wide unaligned global accesses)
template <typename T, int N> __device__ __forceinline__ void load_n(const T *p, float (&f)[N])
{
    T v[N];
    __builtin_memcpy(v, p, N * sizeof(T));
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = (float)v[j];
}
template <typename T, int N> __device__ __forceinline__ void store_n(T *p, const float (&f)[N])
{
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)f[j]; // to nearest even
    __builtin_memcpy(p, v, N * sizeof(T));
}
__device__ __forceinline__ float load_w(const void *w, int dtype, int i)
{
    if (dtype == BFA_F32) return ((const float *)w)[i];
    if (dtype == BFA_F16) return (float)((const _Float16 *)w)[i];
    return (float)((const __bf16 *)w)[i];
}
// N of them from i on; no weights: `none`
template <int N> __device__ __forceinline__ void load_w_n(const void *w, int dtype, int i, float none, float (&f)[N])
{
    if (!w) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = none;
    } else if (dtype == BFA_F32) load_n<float, N>((const float *)w + i, f);
    else if (dtype == BFA_F16) load_n<_Float16, N>((const _Float16 *)w + i, f);
    else load_n<__bf16, N>((const __bf16 *)w + i, f);
}
__device__ __forceinline__ void store_w(void *w, int dtype, int i, float v)
{
    if (dtype == BFA_F32) ((float *)w)[i] = v;
    else if (dtype == BFA_F16) ((_Float16 *)w)[i] = (_Float16)v;
    else ((__bf16 *)w)[i] = (__bf16)v;
}

template <int CTRL> __device__ __forceinline__ float dpp_f(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ int dpp_i(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ double dpp_d(double x)
{
    const long long v = __double_as_longlong(x);
    const unsigned lo = (unsigned)dpp_i<CTRL>((int)(unsigned)v), hi = (unsigned)dpp_i<CTRL>((int)(v >> 32));
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
constexpr int DPP_QUAD_X1 = 0xB1, DPP_QUAD_X2 = 0x4E;             // lane ^ 1, lane ^ 2
constexpr int DPP_ROR = 0x120, DPP_SHR = 0x110;                   // row_ror:n, row_shr:n inside 16 lanes

struct OpAdd { template <typename V> static __device__ __forceinline__ V f(V a, V b) { return a + b; } };
struct OpMax { template <typename V> static __device__ __forceinline__ V f(V a, V b) { return a > b ? a : b; }
               static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); } };
struct OpMin { template <typename V> static __device__ __forceinline__ V f(V a, V b) { return a < b ? a : b; }
               static __device__ __forceinline__ float f(float a, float b) { return fminf(a, b); } };
template <int CTRL> __device__ __forceinline__ float dpp(float x) { return dpp_f<CTRL>(x); }
template <int CTRL> __device__ __forceinline__ int dpp(int x) { return dpp_i<CTRL>(x); }
template <int CTRL> __device__ __forceinline__ double dpp(double x) { return dpp_d<CTRL>(x); }
template <int CTRL> __device__ __forceinline__ unsigned long long dpp(unsigned long long x)
{
    const unsigned lo = (unsigned)dpp_i<CTRL>((int)(unsigned)x), hi = (unsigned)dpp_i<CTRL>((int)(x >> 32));
    return ((unsigned long long)hi << 32) | lo;
}

// the reduction over the aligned group of G = 4, 16 or 64 lanes, in every lane of the group.  All lanes of a group are active or none.
template <int G, typename Op, typename V> __device__ __forceinline__ V group_all(V x)
{
    static_assert(G == 4 || G == 16 || G == 64, "");
    if constexpr (G == 4) {
        x = Op::f(x, dpp<DPP_QUAD_X1>(x));
        x = Op::f(x, dpp<DPP_QUAD_X2>(x));
    } else {
        x = Op::f(x, dpp<DPP_ROR + 8>(x));
        x = Op::f(x, dpp<DPP_ROR + 4>(x));
        x = Op::f(x, dpp<DPP_ROR + 2>(x));
        x = Op::f(x, dpp<DPP_ROR + 1>(x));
        if constexpr (G == 64) {
            x = Op::f(x, __shfl_xor(x, 16));
            x = Op::f(x, __shfl_xor(x, 32));
        }
    }
    return x;
}

// the reduction over the W waves of a workgroup (all threads call it, all get the result; waves are combined in order).
// `sm` has 2 * W entries; `turn` flips between calls so that one barrier per call is enough.
template <int W, typename Op, typename V> __device__ __forceinline__ V block_all(V x, V *sm, int &turn)
{
    x = group_all<64, Op>(x);
    if constexpr (W > 1) {
        V *s = sm + (turn ? W : 0);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
        __syncthreads();
        x = s[0];
#pragma unroll
        for (int k = 1; k < W; ++k) x = Op::f(x, s[k]);
    }
    return x;
}

// e^x for x <= 0 with a relative error of about 2^-23 also where x is large: x log2(e) in two parts, the low one as a factor
__device__ __forceinline__ float exp_neg(float x)
{
    const float L2E = 1.44269504f;
    const float hi = x * L2E;
    const float lo = __builtin_fmaf(x, L2E, -hi);
    const float e = __builtin_amdgcn_exp2f(hi);
    return hi < -150.0f ? 0.0f : __builtin_fmaf(e, lo * 0.693147181f, e); // (-inf gives 0, NaN stays)
}
#endif

} // namespace bfa
