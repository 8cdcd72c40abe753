// bfa_loss.hip -- weighted cross entropy of rows of logits [B, T, C] against one label per row, with its gradient.
//
//   m = max z,  s = sum exp(z - m),  nll = m + log s - z[label]
//   none: w nll per row;   sum: sum w nll;   mean: sum w nll / sum w   (0 where sum w is 0)
//   dz = u w (exp(z - m) / s - onehot(label))   with u = grad_scale * upstream (/ sum w for the mean)
//
// A row counts when t < T_len[b], its label is not negative and its weight not 0; the others give 0 and dz = 0 and are not read.  A label >= C
// gives NaN in that row.
//
// Bound: HBM.  One kernel does loss and gradient: it reads a row once, keeps it in registers (as stored, so 16-bit logits take
// half a register), and writes the gradient from there, so the path moves its logits once in and its gradient once out.  The same
// kernel without the gradient is the forward pass, and without the loss the backward pass of a loss whose upstream gradient was
// not known: recomputing max and sum from the row in registers costs less than keeping them.  Exponentials and sums are float32.
// sum w (one pass over the labels, before) and the sum of the losses (after) are float64 partial sums per workgroup, added in a
// fixed order: no atomics.
#include <algorithm>

#include "bfa_rows.hpp"

namespace bfa {

struct LossArgs {
    RowShape s;
    RowPtr z, dz;            // dz.p null: no gradient
    const int32_t *labels;   // [B, T]
    const float *weights;    // [B, T] or null
    const float *up;         // upstream gradient: [B, T] for `none`, one number otherwise; null: 1
    const double *wsum;      // `mean`: partial sums of the weights
    int n_wsum;
    int per_row;             // `none`
    float scale;
    float *nll;              // `none`: [B, T] or null
    double *part;            // otherwise: [gridDim.x] or null
};

// what of a row is needed besides its logits; the loss of a row counts with weight w, its gradient with g
struct RowWeight { int label; float w, g; };
__device__ __forceinline__ RowWeight row_weight(const LossArgs &a, uint32_t r, uint32_t b, uint32_t t, float scale)
{
    RowWeight q = {-1, 0.0f, 0.0f};
    if (!a.s.held(b, t)) return q;
    q.label = a.labels[r];
    if (q.label < 0) { q.label = -1; return q; }
    q.w = a.weights ? a.weights[r] : 1.0f;
    if (q.w == 0.0f) { q.label = -1; return q; }
    q.g = q.w * scale;
    if (a.per_row && a.up) q.g *= a.up[r];
    return q;
}
// the factor all rows share; every thread of the workgroup gets it
__device__ __forceinline__ float shared_scale(const LossArgs &a)
{
    float u = a.scale;
    if (!a.per_row && a.up) u *= a.up[0];
    if (a.wsum) {
        double s = 0.0;
        for (int i = 0; i < a.n_wsum; ++i) s += a.wsum[i];
        u = s == 0.0 ? 0.0f : (float)((double)u / s);
    }
    return u;
}

// partial sums of the weights of the rows that count
__global__ __launch_bounds__(256) void k_loss_weights(LossArgs a, double *out)
{
    __shared__ double sm[8];
    int turn = 0;
    double s = 0.0;
    for (uint32_t r = blockIdx.x * 256 + threadIdx.x; r < a.s.rows; r += gridDim.x * 256) {
        uint32_t b, t;
        a.s.split(r, b, t);
        s += (double)row_weight(a, r, b, t, 0.0f).w;
    }
    s = block_all<4, OpAdd>(s, sm, turn);
    if (threadIdx.x == 0) out[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void k_loss_finish(const double *part, int n, const double *wsum, int n_wsum, float *out)
{
    __shared__ double sm[8];
    int turn = 0;
    double s = 0.0, w = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    for (int i = threadIdx.x; i < n_wsum; i += 256) w += wsum[i];
    s = block_all<4, OpAdd>(s, sm, turn);
    w = block_all<4, OpAdd>(w, sm, turn);
    if (threadIdx.x == 0) out[0] = wsum ? (w == 0.0 ? 0.0f : (float)(s / w)) : (float)s;
}

// Short rows (C <= 512): G lanes share a row, each has E = ceil(C / G) consecutive elements; the last chunk is moved back to end
// with the row and its elements that belong to the chunk before it do not count twice.
template <typename T, int G, int E> __global__ __launch_bounds__(256) void k_loss_short(LossArgs a)
{
    __shared__ double sm[8];
    constexpr int RPG = 256 / G;
    const int l = threadIdx.x % G, C = a.s.C;
    const int first = l * E, at = min(first, C - E);
    const bool on = first < C;
    const float scale = a.dz.p ? shared_scale(a) : 0.0f;
    double sum = 0.0;
    for (uint32_t r = blockIdx.x * RPG + threadIdx.x / G; r < a.s.rows; r += gridDim.x * RPG) {
        uint32_t b, t;
        a.s.split(r, b, t);
        const RowWeight q = row_weight(a, r, b, t, scale);
        float e[E], nll = 0.0f;
        if (q.label >= 0) { // (the same for the G lanes of a row)
            const T *z = row_in<T>(a.z, b, t);
            load_n<T, E>(z + at, e);
            const float zl = (float)z[min(q.label, C - 1)];
            float m = e[0], s = 0.0f;
#pragma unroll
            for (int j = 1; j < E; ++j) m = fmaxf(m, e[j]);
            m = group_all<G, OpMax>(m);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                e[j] = exp_neg(e[j] - m);
                s += (on && at + j >= first) ? e[j] : 0.0f;
            }
            s = group_all<G, OpAdd>(s);
            const bool bad = q.label >= C;
            nll = bad ? __builtin_nanf("") : q.w * (logf(s) + (m - zl));
            const float g = bad ? __builtin_nanf("") : q.g, p = g / s;
#pragma unroll
            for (int j = 0; j < E; ++j) e[j] = e[j] * p - (at + j == q.label ? g : 0.0f);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) e[j] = 0.0f;
        }
        if (a.dz.p && on) store_n<T, E>(row_out<T>(a.dz, b, t) + at, e);
        if (l == 0) {
            if (a.nll) a.nll[r] = nll;
            sum += (double)nll;
        }
    }
    if (a.part) {
        int turn = 0;
        sum = block_all<4, OpAdd>(sum, sm, turn);
        if (threadIdx.x == 0) a.part[blockIdx.x] = sum;
    }
}

// Long rows: a workgroup of TPR threads per row (TPR = 64: four rows per workgroup, a wave each), NH 16-byte vectors per thread
// held in registers as stored; what a row has beyond TPR * NH vectors (vocabularies of more than 131072 16-bit or 65536 float32
// classes) is read again for each of the three sweeps, from the caches.
template <typename T, int TPR, int NH> __global__ __launch_bounds__(TPR <= 256 ? 256 : TPR) void k_loss_long(LossArgs a)
{
    constexpr int VEC = 16 / sizeof(T), WG = TPR <= 256 ? 256 : TPR, RPG = WG / TPR, W = TPR / 64;
    __shared__ float sm[2 * W];
    __shared__ double smd[2 * (WG / 64)];
    const int l = threadIdx.x % TPR, C = a.s.C;
    const int held_end = min(C, TPR * NH * VEC);
    int turn = 0;
    const float scale = a.dz.p ? shared_scale(a) : 0.0f;
    double sum = 0.0;
    struct Vec { T v[VEC]; };
    for (uint32_t r = blockIdx.x * RPG + threadIdx.x / TPR; r < a.s.rows; r += gridDim.x * RPG) {
        uint32_t b, t;
        a.s.split(r, b, t);
        const RowWeight q = row_weight(a, r, b, t, scale);
        T *dz = a.dz.p ? row_out<T>(a.dz, b, t) : nullptr;
        float nll = 0.0f;
        if (q.label >= 0) { // (the same for the threads of a row)
            const T *z = row_in<T>(a.z, b, t);
            Vec x[NH];
#pragma unroll
            for (int v = 0; v < NH; ++v) {
                const int i = (v * TPR + l) * VEC;
                if (i < C) __builtin_memcpy(&x[v], z + min(i, C - VEC), 16);
            }
            float m = -__builtin_inff();
#pragma unroll
            for (int v = 0; v < NH; ++v)
                if ((v * TPR + l) * VEC < C) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) m = fmaxf(m, (float)x[v].v[j]);
                }
            for (int i = held_end + l; i < C; i += TPR) m = fmaxf(m, (float)z[i]);
            if constexpr (W == 1) m = group_all<64, OpMax>(m); else m = block_all<W, OpMax>(m, sm, turn);
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < NH; ++v) {
                const int i = (v * TPR + l) * VEC;
                if (i < C) {
                    const int skip = max(i - (C - VEC), 0); // elements of a vector moved back that the one before it has counted
#pragma unroll
                    for (int j = 0; j < VEC; ++j) s += j >= skip ? exp_neg((float)x[v].v[j] - m) : 0.0f;
                }
            }
            for (int i = held_end + l; i < C; i += TPR) s += exp_neg((float)z[i] - m);
            if constexpr (W == 1) s = group_all<64, OpAdd>(s); else s = block_all<W, OpAdd>(s, sm, turn);
            const bool bad = q.label >= C;
            nll = bad ? __builtin_nanf("") : q.w * (logf(s) + (m - (float)z[min(q.label, C - 1)]));
            if (dz) {
                const float g = bad ? __builtin_nanf("") : q.g, p = g / s;
#pragma unroll
                for (int v = 0; v < NH; ++v) {
                    const int i = (v * TPR + l) * VEC;
                    if (i < C) {
                        const int at = min(i, C - VEC);
                        float o[VEC];
#pragma unroll
                        for (int j = 0; j < VEC; ++j) o[j] = exp_neg((float)x[v].v[j] - m) * p - (at + j == q.label ? g : 0.0f);
                        store_n<T, VEC>(dz + at, o);
                    }
                }
                for (int i = held_end + l; i < C; i += TPR) dz[i] = (T)(exp_neg((float)z[i] - m) * p - (i == q.label ? g : 0.0f));
            }
        } else if (dz) {
            const float o[VEC] = {};
            for (int i = l * VEC; i < C; i += TPR * VEC) store_n<T, VEC>(dz + min(i, C - VEC), o);
        }
        if (l == 0) {
            if (a.nll) a.nll[r] = nll;
            sum += (double)nll;
        }
    }
    if (a.part) {
        int turnd = 0;
        sum = block_all<WG / 64, OpAdd>(sum, smd, turnd);
        if (threadIdx.x == 0) a.part[blockIdx.x] = sum;
    }
}

constexpr int LOSS_MAX_GRID = 2048, LOSS_WSUM = 256;

template <typename T, int G, int E> static int loss_short(const LossArgs &a, hipStream_t st)
{
    const int grid = (int)std::min<uint32_t>((a.s.rows + 256 / G - 1) / (256 / G), LOSS_MAX_GRID);
    hipLaunchKernelGGL((k_loss_short<T, G, E>), dim3(grid), dim3(256), 0, st, a);
    return grid;
}
template <typename T, int G> static int loss_short_e(const LossArgs &a, hipStream_t st)
{
    switch ((a.s.C + G - 1) / G) {
    case 1: return loss_short<T, G, 1>(a, st);
    case 2: return loss_short<T, G, 2>(a, st);
    case 3: return loss_short<T, G, 3>(a, st);
    case 4: return loss_short<T, G, 4>(a, st);
    case 5: return loss_short<T, G, 5>(a, st);
    case 6: return loss_short<T, G, 6>(a, st);
    case 7: return loss_short<T, G, 7>(a, st);
    default: return loss_short<T, G, 8>(a, st);
    }
}
template <typename T, int TPR, int NH> static int loss_long(const LossArgs &a, hipStream_t st)
{
    constexpr int WG = TPR <= 256 ? 256 : TPR, RPG = WG / TPR;
    const int grid = (int)std::min<uint32_t>((a.s.rows + RPG - 1) / RPG, 256 * 2048 / WG);
    hipLaunchKernelGGL((k_loss_long<T, TPR, NH>), dim3(grid), dim3(WG), 0, st, a);
    return grid;
}
// -> the workgroups launched (entries of a.part)
template <typename T> static int loss_launch(const LossArgs &a, hipStream_t st)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    const int C = a.s.C;
    if (C <= 32) return loss_short_e<T, 4>(a, st);
    if (C <= 128) return loss_short_e<T, 16>(a, st);
    if (C <= 512) return loss_short_e<T, 64>(a, st);
    if (C <= 64 * 4 * VEC) return loss_long<T, 64, 4>(a, st);
    if (C <= 256 * 4 * VEC) return loss_long<T, 256, 4>(a, st);
    if (C <= 1024 * 4 * VEC) return loss_long<T, 1024, 4>(a, st);
    if (C <= 1024 * 8 * VEC) return loss_long<T, 1024, 8>(a, st);
    return loss_long<T, 1024, 16>(a, st);
}

} // namespace bfa

extern "C" size_t bfa_loss_ws_doubles() { return bfa::LOSS_WSUM + bfa::LOSS_MAX_GRID; }

// reduction: 0 none, 1 sum, 2 mean.  out: [B, T] for none, one number otherwise, or null.  dz or null.
extern "C" int bfa_launch_loss(const bfa_rows *z, int B, int T, int C, const int32_t *T_len, const int32_t *labels, const float *weights,
                               int reduction, float scale, const float *up, float *out, const bfa_rows *dz, double *ws, void *stream)
{
    using namespace bfa;
    hipStream_t st = (hipStream_t)stream;
    LossArgs a{RowShape(B, T, C, T_len), {z->data, z->strideB, z->strideT}, {dz ? dz->data : nullptr, dz ? dz->strideB : 0, dz ? dz->strideT : 0},
               labels, weights, up, nullptr, 0, reduction == 0, scale, reduction == 0 ? out : nullptr, nullptr};
    if (reduction == 2) {
        a.n_wsum = (int)std::min<uint32_t>((a.s.rows + 2047) / 2048, LOSS_WSUM);
        hipLaunchKernelGGL(k_loss_weights, dim3(a.n_wsum), dim3(256), 0, st, a, ws);
        a.wsum = ws;
    }
    if (reduction != 0 && out) a.part = ws + LOSS_WSUM;
    int grid = 0;
    if (a.s.rows == 0) grid = 0; // (the loss of no rows: the last kernel alone)
    else if (z->dtype == BFA_F32) grid = loss_launch<float>(a, st);
    else if (z->dtype == BFA_F16) grid = loss_launch<_Float16>(a, st);
    else grid = loss_launch<__bf16>(a, st);
    if (a.part) hipLaunchKernelGGL(k_loss_finish, dim3(1), dim3(256), 0, st, a.part, grid, a.wsum, a.n_wsum, out);
    return (int)hipGetLastError();
}
