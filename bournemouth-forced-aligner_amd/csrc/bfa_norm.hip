// bfa_norm.hip -- layer normalisation of rows [B, T, C] and its backward pass.
//
//   y = xh w + b,  xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Rows behind T_len[b] are not read: y = 0, mean = rstd = 0, dx = 0, and nothing of them goes into dw / db.
//
// Bound: HBM.  A row is read once and stays in the registers of the TPR threads that share it (at most 16 elements each), so
// the variance is the two-pass one (deviations from the mean, float32) at no extra traffic, and the mean's own rounding is taken
// from the deviations again (norm_stat).  The last 16-byte vector of a row is
// moved back to end with the row where C is not a multiple of it -- wide loads and stores for every C and every alignment; the
// elements it shares with its neighbour are counted once (`own`) and stored twice with the same value.
// Workgroups stride over the rows: the weights are loaded once per workgroup, and in the backward pass a thread keeps the sums
// of its own columns in registers.  Per workgroup one partial sum per column goes to the workspace, and k_norm_cols adds those
// in a fixed order: no atomics, the same bits every time.
//
// Measured: 32768 rows of 4096 bfloat16 channels 104-107 us forward (5.0-5.2 TB/s; 100 without the correction of the mean), 171 us
// backward (4.7 TB/s) + 6.6 for the column sums; 16 ragged utterances of up to 1870 x 768 float32 24 + 35 + 5 us; 12000 ragged rows of 1001
// float16 channels, every row at another alignment, 11 + 15 + 6 us (35 + 21 with the weights loaded one by one).
// 8192 rows of 8192 / 16384 bfloat16 channels 60 / 122-126 us forward (4.5 / 4.4 TB/s), 122 + 7 / 203 + 14 us backward (3.3 / 4.0 TB/s:
// x, dy, w and the two sums as floats, 7 to 16 vector registers spilled); of 20480, swept element by element, 430 us and 662 + 266 + 6 us.
#include <algorithm>

#include "bfa_rows.hpp"

namespace bfa {

struct NormArgs {
    RowShape s;
    RowPtr x, y, dy; // forward: x -> y; backward: dy, x -> y (dx)
    const void *w, *b;
    int wtype;
    float eps;
    float *mean, *rstd;
    float *part; // backward: [gridDim.x][2][C] or null
};

template <int TPR> struct NormGeo {
    static constexpr int WG = TPR <= 256 ? 256 : TPR;
    static constexpr int RPG = WG / TPR; // rows a workgroup works on at a time
    static constexpr int W = TPR <= 64 ? 1 : TPR / 64;
};

template <int TPR> __device__ __forceinline__ float norm_sum(float v, float *sm, int &turn)
{
    if constexpr (TPR <= 64) return group_all<TPR, OpAdd>(v);
    else return block_all<TPR / 64, OpAdd>(v, sm, turn);
}
// the sums of two numbers behind one barrier (sm: 4 * W entries)
template <int TPR> __device__ __forceinline__ void norm_sum2(float &a, float &b, float *sm, int &turn)
{
    constexpr int W = TPR / 64;
    a = group_all<(TPR < 64 ? TPR : 64), OpAdd>(a);
    b = group_all<(TPR < 64 ? TPR : 64), OpAdd>(b);
    if constexpr (W > 1) {
        float *s = sm + (turn ? 2 * W : 0);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) { s[threadIdx.x >> 6] = a; s[W + (threadIdx.x >> 6)] = b; }
        __syncthreads();
        a = s[0];
        b = s[W];
#pragma unroll
        for (int k = 1; k < W; ++k) { a += s[k]; b += s[W + k]; }
    }
}
// Mean and rstd of a row from its deviations from a first mean m (their sum and the sum of their squares).  The deviations of a row whose
// mean is large against its spread are exact, the mean itself is rounded: what it lacks, `shift`, is the deviations' mean.
struct NormStat { float shift, rstd; };
__device__ __forceinline__ NormStat norm_stat(float sum, float squares, float inv_c, float eps)
{
    const float shift = sum * inv_c, var = squares * inv_c - shift * shift;
    return {shift, 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps)}; // (NaN stays)
}

template <typename T, int VEC, int TPR, int NV>
__global__ __launch_bounds__(NormGeo<TPR>::WG) void k_norm(NormArgs a)
{
    using Geo = NormGeo<TPR>;
    __shared__ float sm[4 * Geo::W];
    const int l = threadIdx.x % TPR, C = a.s.C;
    const float inv_c = 1.0f / (float)C;
    int turn = 0;
    int at[NV];
    float w[NV][VEC], b[NV][VEC];
    const int last = ((NV - 1) * TPR + l) * VEC; // where this thread's last vector would start
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        at[v] = min((v * TPR + l) * VEC, C - VEC);
        load_w_n<VEC>(a.w, a.wtype, at[v], 1.0f, w[v]);
        load_w_n<VEC>(a.b, a.wtype, at[v], 0.0f, b[v]);
    }
    auto own = [&](int v, int j) { return v < NV - 1 || (last < C && at[v] + j >= last); };
    for (uint32_t r = blockIdx.x * Geo::RPG + threadIdx.x / TPR; r < a.s.rows; r += gridDim.x * Geo::RPG) {
        uint32_t bb, t;
        a.s.split(r, bb, t);
        T *y = row_out<T>(a.y, bb, t);
        float x[NV][VEC], mean = 0.0f, rstd = 0.0f;
        if (a.s.held(bb, t)) { // (the same for the TPR threads of a row)
            const T *px = row_in<T>(a.x, bb, t);
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) load_n<T, VEC>(px + at[v], x[v]);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += own(v, j) ? x[v][j] : 0.0f;
            mean = norm_sum<TPR>(s, sm, turn) / (float)C;
            float q = 0.0f;
            s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    x[v][j] -= mean;
                    s += own(v, j) ? x[v][j] : 0.0f;
                    q = own(v, j) ? __builtin_fmaf(x[v][j], x[v][j], q) : q;
                }
            norm_sum2<TPR>(s, q, sm, turn);
            const NormStat st = norm_stat(s, q, inv_c, a.eps);
            rstd = st.rstd;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[v][j] = __builtin_fmaf((x[v][j] - st.shift) * rstd, w[v][j], b[v][j]);
            mean += st.shift;
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[v][j] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v < NV - 1 || last < C) store_n<T, VEC>(y + at[v], x[v]);
        if (l == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T, int VEC, int TPR, int NV>
__global__ __launch_bounds__(NormGeo<TPR>::WG) void k_norm_bwd(NormArgs a)
{
    using Geo = NormGeo<TPR>;
    __shared__ float sm[2 * Geo::W];
    const int l = threadIdx.x % TPR, C = a.s.C;
    const float inv_c = 1.0f / (float)C;
    int turn = 0;
    int at[NV];
    float w[NV][VEC], sw[NV][VEC], sb[NV][VEC];
    const int last = ((NV - 1) * TPR + l) * VEC;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        at[v] = min((v * TPR + l) * VEC, C - VEC);
        load_w_n<VEC>(a.w, a.wtype, at[v], 1.0f, w[v]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sw[v][j] = sb[v][j] = 0.0f;
    }
    auto own = [&](int v, int j) { return v < NV - 1 || (last < C && at[v] + j >= last); };
    for (uint32_t r = blockIdx.x * Geo::RPG + threadIdx.x / TPR; r < a.s.rows; r += gridDim.x * Geo::RPG) {
        uint32_t bb, t;
        a.s.split(r, bb, t);
        float x[NV][VEC];
        if (a.s.held(bb, t)) {
            const T *px = row_in<T>(a.x, bb, t), *pd = row_in<T>(a.dy, bb, t);
            const float mean = a.mean[r], rstd = a.rstd[r];
            float d[NV][VEC], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) { load_n<T, VEC>(px + at[v], x[v]); load_n<T, VEC>(pd + at[v], d[v]); }
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    x[v][j] = (x[v][j] - mean) * rstd;
                    sw[v][j] = __builtin_fmaf(d[v][j], x[v][j], sw[v][j]);
                    sb[v][j] += d[v][j];
                    d[v][j] *= w[v][j];
                    s1 += own(v, j) ? d[v][j] : 0.0f;
                    s2 = own(v, j) ? __builtin_fmaf(d[v][j], x[v][j], s2) : s2;
                }
            s1 = norm_sum<TPR>(s1, sm, turn) * inv_c;
            s2 = norm_sum<TPR>(s2, sm, turn) * inv_c;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[v][j] = rstd * (d[v][j] - s1 - x[v][j] * s2);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[v][j] = 0.0f;
        }
        if (a.y.p) {
            T *dx = row_out<T>(a.y, bb, t);
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (v < NV - 1 || last < C) store_n<T, VEC>(dx + at[v], x[v]);
        }
    }
    if (!a.part) return;
    float *pw = a.part + (int64_t)blockIdx.x * 2 * C;
    if constexpr (Geo::RPG == 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (own(v, j)) { pw[at[v] + j] = sw[v][j]; pw[C + at[v] + j] = sb[v][j]; }
    } else { // the RPG rows of the workgroup meet in LDS, in order
        __shared__ float acc[Geo::RPG][TPR * NV * VEC];
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (own(v, j)) acc[threadIdx.x / TPR][at[v] + j] = k ? sb[v][j] : sw[v][j];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += Geo::WG) {
                float s = acc[0][c];
#pragma unroll
                for (int g = 1; g < Geo::RPG; ++g) s += acc[g][c];
                pw[k * C + c] = s;
            }
        }
    }
}

// rows longer than the registers of a workgroup hold: 1024 threads sweep the row three times (the second and third time it
// comes from the caches)
template <typename T> __global__ __launch_bounds__(1024) void k_norm_long(NormArgs a)
{
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float sm[64];
    const int C = a.s.C, n = C / VEC * VEC;
    int turn = 0;
    for (uint32_t r = blockIdx.x; r < a.s.rows; r += gridDim.x) {
        uint32_t bb, t;
        a.s.split(r, bb, t);
        T *y = row_out<T>(a.y, bb, t);
        float mean = 0.0f, shift = 0.0f, rstd = 0.0f;
        const bool held = a.s.held(bb, t);
        const T *px = row_in<T>(a.x, bb, t);
        if (held) {
            float s = 0.0f, x[VEC];
            for (int i = threadIdx.x * VEC; i < n; i += 1024 * VEC) {
                load_n<T, VEC>(px + i, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += x[j];
            }
            if (n + (int)threadIdx.x < C) s += (float)px[n + threadIdx.x];
            mean = norm_sum<1024>(s, sm, turn) / (float)C;
            float q = 0.0f;
            s = 0.0f;
            for (int i = threadIdx.x * VEC; i < n; i += 1024 * VEC) {
                load_n<T, VEC>(px + i, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { const float d = x[j] - mean; s += d; q = __builtin_fmaf(d, d, q); }
            }
            if (n + (int)threadIdx.x < C) { const float d = (float)px[n + threadIdx.x] - mean; s += d; q = __builtin_fmaf(d, d, q); }
            norm_sum2<1024>(s, q, sm, turn);
            const NormStat st = norm_stat(s, q, 1.0f / (float)C, a.eps);
            shift = st.shift;
            rstd = st.rstd;
        }
        for (int i = threadIdx.x; i < C; i += 1024) {
            const float v = held ? __builtin_fmaf((((float)px[i] - mean) - shift) * rstd, a.w ? load_w(a.w, a.wtype, i) : 1.0f,
                                                  a.b ? load_w(a.b, a.wtype, i) : 0.0f) : 0.0f;
            y[i] = (T)v;
        }
        mean += shift;
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T> __global__ __launch_bounds__(1024) void k_norm_bwd_long(NormArgs a)
{
    __shared__ float sm[32];
    const int C = a.s.C;
    int turn = 0;
    for (uint32_t r = blockIdx.x; r < a.s.rows; r += gridDim.x) {
        uint32_t bb, t;
        a.s.split(r, bb, t);
        const bool held = a.s.held(bb, t);
        const T *px = row_in<T>(a.x, bb, t), *pd = row_in<T>(a.dy, bb, t);
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        if (held) {
            for (int i = threadIdx.x; i < C; i += 1024) {
                const float g = (float)pd[i] * (a.w ? load_w(a.w, a.wtype, i) : 1.0f);
                s1 += g;
                s2 = __builtin_fmaf(g, ((float)px[i] - mean) * rstd, s2);
            }
            s1 = block_all<16, OpAdd>(s1, sm, turn) / (float)C;
            s2 = block_all<16, OpAdd>(s2, sm, turn) / (float)C;
        }
        T *dx = row_out<T>(a.y, bb, t);
        for (int i = threadIdx.x; i < C; i += 1024)
            dx[i] = (T)(held ? rstd * ((float)pd[i] * (a.w ? load_w(a.w, a.wtype, i) : 1.0f) - s1 - ((float)px[i] - mean) * rstd * s2) : 0.0f);
    }
}

// the column sums of such rows: a thread per column, blockIdx.y takes every gridDim.y-th row
template <typename T> __global__ __launch_bounds__(256) void k_norm_colsum_long(NormArgs a)
{
    const int c = blockIdx.x * 256 + threadIdx.x, C = a.s.C;
    if (c >= C) return;
    float sw = 0.0f, sb = 0.0f;
    for (uint32_t r = blockIdx.y; r < a.s.rows; r += gridDim.y) {
        uint32_t bb, t;
        a.s.split(r, bb, t);
        if (!a.s.held(bb, t)) continue;
        const float d = (float)row_in<T>(a.dy, bb, t)[c];
        sw = __builtin_fmaf(d, ((float)row_in<T>(a.x, bb, t)[c] - a.mean[r]) * a.rstd[r], sw);
        sb += d;
    }
    float *pw = a.part + (int64_t)blockIdx.y * 2 * C;
    pw[c] = sw;
    pw[C + c] = sb;
}

// dw / db from the workgroups' partial sums [n][2][C]: 64 columns of the 2 C per workgroup, 16 ranges of the n added side by
// side and then in order
__global__ __launch_bounds__(1024) void k_norm_cols(const float *part, int n, int C, void *dw, void *db, int wtype)
{
    __shared__ float sm[16][64];
    const int l = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + l, width = 2 * (int64_t)C;
    float s = 0.0f;
    if (c < width) {
        const int per = (n + 15) / 16, i1 = min(n, (q + 1) * per);
#pragma unroll 8
        for (int i = q * per; i < i1; ++i) s += part[i * width + c];
    }
    sm[q][l] = s;
    __syncthreads();
    if (q == 0 && c < width) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += sm[k][l];
        if (c < C) { if (dw) store_w(dw, wtype, (int)c, s); }
        else if (db) store_w(db, wtype, (int)(c - C), s);
    }
}

// rows of at most 16384 elements are held in registers: the fewest threads of 16 / 64 / 256 / 1024 with at most 16 elements each
constexpr int NORM_MAX_HELD = 16384;
// workgroups of the backward pass (each leaves one partial sum per column)
static int norm_bwd_grid(uint32_t rows, int C)
{
    const int tpr = C <= 256 ? 16 : C <= 1024 ? 64 : C <= 4096 ? 256 : 1024;
    if (C > NORM_MAX_HELD) return (int)std::min<uint32_t>(rows, 64);
    const int rpg = tpr <= 256 ? 256 / tpr : 1;
    const uint32_t groups = (rows + rpg - 1) / rpg;
    return (int)std::min<uint32_t>(groups, tpr == 1024 ? 512 : 1024);
}

template <typename T, int TPR, int NV, int VEC = 16 / (int)sizeof(T)> static void norm_go(const NormArgs &a, bool bwd, hipStream_t st)
{
    using Geo = NormGeo<TPR>;
    const uint32_t groups = (a.s.rows + Geo::RPG - 1) / Geo::RPG;
    if (bwd) hipLaunchKernelGGL((k_norm_bwd<T, VEC, TPR, NV>), dim3((unsigned)norm_bwd_grid(a.s.rows, a.s.C)), dim3(Geo::WG), 0, st, a);
    else hipLaunchKernelGGL((k_norm<T, VEC, TPR, NV>), dim3(std::min<uint32_t>(groups, 256u * 2048 / Geo::WG)), dim3(Geo::WG), 0, st, a);
}

template <typename T, int TPR> static void norm_nv(const NormArgs &a, bool bwd, hipStream_t st)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const int nv = (a.s.C + TPR * VEC - 1) / (TPR * VEC);
    if (nv <= 1) norm_go<T, TPR, 1>(a, bwd, st);
    else if (nv == 2) norm_go<T, TPR, 2>(a, bwd, st);
    else if constexpr (VEC == 4) {
        if (nv == 3) norm_go<T, TPR, 3>(a, bwd, st);
        else norm_go<T, TPR, 4>(a, bwd, st);
    }
}

template <typename T> static void norm_launch(const NormArgs &a, bool bwd, hipStream_t st)
{
    const int C = a.s.C;
    if (C < 16 / (int)sizeof(T)) norm_go<T, 16, 1, 1>(a, bwd, st); // shorter than a vector: element by element
    else if (C <= 256) norm_nv<T, 16>(a, bwd, st);
    else if (C <= 1024) norm_nv<T, 64>(a, bwd, st);
    else if (C <= 4096) norm_nv<T, 256>(a, bwd, st);
    else if (C <= NORM_MAX_HELD) norm_nv<T, 1024>(a, bwd, st);
    else if (!bwd) hipLaunchKernelGGL((k_norm_long<T>), dim3(std::min<uint32_t>(a.s.rows, 512)), dim3(1024), 0, st, a);
    else {
        if (a.y.p) hipLaunchKernelGGL((k_norm_bwd_long<T>), dim3(std::min<uint32_t>(a.s.rows, 512)), dim3(1024), 0, st, a);
        if (a.part)
            hipLaunchKernelGGL((k_norm_colsum_long<T>), dim3((unsigned)((C + 255) / 256), (unsigned)norm_bwd_grid(a.s.rows, C)), dim3(256), 0, st, a);
    }
}

} // namespace bfa

extern "C" size_t bfa_norm_ws_floats(int B, int T, int C)
{
    return (size_t)bfa::norm_bwd_grid((uint32_t)((int64_t)B * T), C) * 2 * (size_t)C;
}

extern "C" int bfa_launch_norm(int dtype, const bfa_rows *x, int B, int T, int C, const int32_t *T_len, const void *w, const void *b,
                               int wtype, float eps, const bfa_rows *y, float *mean, float *rstd, void *stream)
{
    using namespace bfa;
    NormArgs a{RowShape(B, T, C, T_len), {x->data, x->strideB, x->strideT}, {y->data, y->strideB, y->strideT}, {nullptr, 0, 0},
               w, b, wtype, eps, mean, rstd, nullptr};
    if (dtype == BFA_F32) norm_launch<float>(a, false, (hipStream_t)stream);
    else if (dtype == BFA_F16) norm_launch<_Float16>(a, false, (hipStream_t)stream);
    else norm_launch<__bf16>(a, false, (hipStream_t)stream);
    return (int)hipGetLastError();
}

extern "C" int bfa_launch_norm_bwd(int dtype, const bfa_rows *dy, const bfa_rows *x, int B, int T, int C, const int32_t *T_len,
                                   const void *w, int wtype, const float *mean, const float *rstd, const bfa_rows *dx, void *dw,
                                   void *db, float *part, void *stream)
{
    using namespace bfa;
    NormArgs a{RowShape(B, T, C, T_len), {x->data, x->strideB, x->strideT}, {dx ? dx->data : nullptr, dx ? dx->strideB : 0, dx ? dx->strideT : 0},
               {dy->data, dy->strideB, dy->strideT}, w, nullptr, wtype, 0.0f, const_cast<float *>(mean), const_cast<float *>(rstd),
               (dw || db) ? part : nullptr};
    if (dtype == BFA_F32) norm_launch<float>(a, true, (hipStream_t)stream);
    else if (dtype == BFA_F16) norm_launch<_Float16>(a, true, (hipStream_t)stream);
    else norm_launch<__bf16>(a, true, (hipStream_t)stream);
    if (dw || db)
        hipLaunchKernelGGL(k_norm_cols, dim3((unsigned)((2 * (int64_t)C + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, part,
                           norm_bwd_grid(a.s.rows, C), C, dw, db, wtype);
    return (int)hipGetLastError();
}
