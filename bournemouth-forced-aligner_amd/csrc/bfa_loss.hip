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
// 4096 x 1000 weighted rows of 67 float32 logits with their gradients: 0.55 ms, 4.1 TB/s.
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
// loaded (for every row of the call, held or not) before it is needed
struct RowAhead {
    int label;
    float w, up;
    __device__ __forceinline__ void load(const LossArgs &a, uint32_t r)
    {
        if (r >= a.s.rows) return;
        label = a.labels[r];
        w = a.weights ? a.weights[r] : 1.0f;
        up = a.per_row && a.up ? a.up[r] : 1.0f;
    }
    __device__ __forceinline__ RowWeight get(const LossArgs &a, uint32_t b, uint32_t t, float scale) const
    {
        if (!a.s.held(b, t) || label < 0 || w == 0.0f) return {-1, 0.0f, 0.0f};
        return {label, w, w * scale * up};
    }
};
__device__ __forceinline__ RowWeight row_weight(const LossArgs &a, uint32_t r, uint32_t b, uint32_t t, float scale)
{
    RowAhead x;
    x.load(a, r);
    return x.get(a, b, t, scale);
}
// the factor all rows share; every thread of the workgroup of W waves calls it and gets it
template <int W> __device__ __forceinline__ float shared_scale(const LossArgs &a, double *sm)
{
    float u = a.scale;
    if (!a.per_row && a.up) u *= a.up[0];
    if (a.wsum) {
        int turn = 0;
        const double s = block_all<W, OpAdd>((int)threadIdx.x < a.n_wsum ? a.wsum[threadIdx.x] : 0.0, sm, turn);
        u = s == 0.0 ? 0.0f : (float)((double)u / s);
        __syncthreads();
    }
    return u;
}

// partial sums of the weights of the rows that count: labels and weights are read four rows at a time
__global__ __launch_bounds__(1024) void k_loss_weights(LossArgs a, double *out)
{
    __shared__ double sm[32];
    int turn = 0;
    double s = 0.0;
    for (uint64_t r0 = ((uint64_t)blockIdx.x * 1024 + threadIdx.x) * 4; r0 < a.s.rows; r0 += (uint64_t)gridDim.x * 4096) {
        int label[4] = {-1, -1, -1, -1};
        float w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        const int n = (int)min((uint64_t)4, a.s.rows - r0);
        if (n == 4) {
            __builtin_memcpy(label, a.labels + r0, 16);
            if (a.weights) __builtin_memcpy(w, a.weights + r0, 16);
        } else {
            for (int j = 0; j < 3; ++j)
                if (j < n) { label[j] = a.labels[r0 + j]; if (a.weights) w[j] = a.weights[r0 + j]; }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bool counts = label[j] >= 0; // (false behind the rows)
            if (a.s.len && counts) {
                uint32_t b, t;
                a.s.split((uint32_t)r0 + j, b, t);
                counts = a.s.held(b, t);
            }
            s += counts ? (double)w[j] : 0.0;
        }
    }
    s = block_all<16, OpAdd>(s, sm, turn);
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
// with the row and its elements that belong to the chunk before it do not count twice.  (Dealt out in turn the lanes of a load lie
// side by side, but there are E of them: 568 us instead of 502 at the time for 4096 x 1000 rows of 67 float32.)  The label and the
// weight of a group's next row are loaded ahead of the work on this one.
template <typename T, int G, int E> __global__ __launch_bounds__(256) void k_loss_short(LossArgs a)
{
    __shared__ double sm[8];
    constexpr int RPG = 256 / G;
    const int l = threadIdx.x % G, C = a.s.C;
    const int first = l * E, at = min(first, C - E);
    const bool on = first < C;
    const float scale = a.dz.p ? shared_scale<4>(a, sm) : 0.0f;
    double sum = 0.0;
    RowAhead ahead;
    uint32_t r = blockIdx.x * RPG + threadIdx.x / G;
    ahead.load(a, r);
    for (; r < a.s.rows; r += gridDim.x * RPG) {
        uint32_t b, t;
        a.s.split(r, b, t);
        const RowWeight q = ahead.get(a, b, t, scale);
        float e[E], nll = 0.0f, zl = 0.0f;
        if (q.label >= 0) { // (the same for the G lanes of a row)
            const T *z = row_in<T>(a.z, b, t);
            load_n<T, E>(z + at, e);
            zl = (float)z[min(q.label, C - 1)];
        }
        ahead.load(a, r + gridDim.x * RPG);
        if (q.label >= 0) {
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

// 16 bytes of a row as stored
template <typename T> struct Packed {
    static constexpr int VEC = 16 / sizeof(T);
    uint32_t u[4];
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(u, p, 16); }
    __device__ __forceinline__ float get(int j) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(u[j]);
        else if constexpr (__is_same(T, __bf16)) return __uint_as_float((j & 1) ? (u[j >> 1] & 0xffff0000u) : (u[j >> 1] << 16));
        else { const uint16_t h = (uint16_t)(u[j >> 1] >> (16 * (j & 1))); return (float)__builtin_bit_cast(_Float16, h); }
    }
    // what was unpacked before is not kept for later (the registers hold the row as stored, not as floats too)
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3])); }
};
// e^x, x <= 0: 16-bit logits take the plain product, which is off by |x| 2^-24 of a weight e^x.  The gradient is rounded to 2^-9 or
// 2^-12 behind it.  In log(sum) it is 2^-24 times the mean |x| under the softmax, at most ln C (7 2^-24 for 131072 normal logits): no more
// than the sum's own additions and the rounding of the loss.  Losses of 131072 bfloat16 and 5003 float16 classes against float64, rms:
// 8.2, 7.2 2^-24 (normal), 3.3 (one class in front), 17.6 (one class 8 to 11 in front of all others alike); by exp_neg 7.9, 7.4, 3.4, 16.5,
// and 1.5 to 14 % slower.
template <typename T> __device__ __forceinline__ float exp_row(float x)
{
    if constexpr (sizeof(T) == 4) return exp_neg(x);
    else return __builtin_amdgcn_exp2f(x * 1.44269504f);
}

// Long rows: a workgroup of TPR threads per row (TPR = 64: four rows per workgroup, a wave each), NH 16-byte vectors per thread
// held in registers as stored; what a row has beyond TPR * NH vectors is read again for each of the three sweeps, from the caches.
// A workgroup strides over rows and fetches the next one's vectors into the registers that the gradient has just been written from.
// 8192 rows of 131072 bfloat16 logits with their gradients: 1.0 ms, 4.3 TB/s (the floats unpacked once and kept spilled: 4.05 ms;
// without the early fetch 1.06; a quarter of the row held, two workgroups per CU, the rest from the caches 1.06).
template <typename T, int TPR, int NH> __global__ __launch_bounds__(TPR <= 256 ? 256 : TPR) void k_loss_long(LossArgs a)
{
    constexpr int VEC = 16 / sizeof(T), WG = TPR <= 256 ? 256 : TPR, RPG = WG / TPR, W = TPR / 64;
    __shared__ float sm[2 * W];
    __shared__ double smd[2 * (WG / 64)];
    const int l = threadIdx.x % TPR, C = a.s.C;
    int turn = 0;
    const float scale = a.dz.p ? shared_scale<WG / 64>(a, smd) : 0.0f;
    double sum = 0.0;
    Packed<T> x[NH];
    RowWeight q;
    const T *z = nullptr;
    auto fetch = [&](int v) {
        const int i = (v * TPR + l) * VEC;
        if (i < C) x[v].load(z + min(i, C - VEC));
    };
    // row r becomes the current one (its vectors are fetched by the caller)
    auto enter = [&](uint32_t r) {
        if (r >= a.s.rows) { q.label = -1; return; }
        uint32_t b, t;
        a.s.split(r, b, t);
        q = row_weight(a, r, b, t, scale);
        z = row_in<T>(a.z, b, t);
    };
    uint32_t r = blockIdx.x * RPG + threadIdx.x / TPR;
    enter(r);
    if (q.label >= 0) {
#pragma unroll
        for (int v = 0; v < NH; ++v) fetch(v);
    }
    while (r < a.s.rows) {
        uint32_t b, t;
        a.s.split(r, b, t);
        T *dz = a.dz.p ? row_out<T>(a.dz, b, t) : nullptr;
        float nll = 0.0f;
        const uint32_t next = r + gridDim.x * RPG;
        bool fetched = false;
        if (q.label >= 0) { // (the same for the threads of a row)
            const float zl = (float)z[min(q.label, C - 1)];
            float m = -__builtin_inff();
            auto max_of = [&](const Packed<T> &p) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) m = fmaxf(m, p.get(j));
            };
#pragma unroll
            for (int v = 0; v < NH; ++v)
                if ((v * TPR + l) * VEC < C) max_of(x[v]);
            // f(the vector, where it would start) for what is not held
            auto beyond = [&](auto &&f) {
                for (int i = (NH * TPR + l) * VEC; i < C; i += 2 * TPR * VEC) {
                    Packed<T> p, p2;
                    const int i2 = i + TPR * VEC;
                    p.load(z + min(i, C - VEC));
                    p2.load(z + min(i2, C - VEC));
                    f(p, i);
                    if (i2 < C) f(p2, i2);
                }
            };
            beyond([&](const Packed<T> &p, int) { max_of(p); });
            if constexpr (W == 1) m = group_all<64, OpMax>(m); else m = block_all<W, OpMax>(m, sm, turn);
            float s = 0.0f;
            auto sum_of = [&](const Packed<T> &p, int i) {
                if (i <= C - VEC) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) s += exp_row<T>(p.get(j) - m);
                } else {
                    const int skip = i - (C - VEC); // elements of a vector moved back that the one before it has counted
#pragma unroll
                    for (int j = 0; j < VEC; ++j) s += j >= skip ? exp_row<T>(p.get(j) - m) : 0.0f;
                }
            };
#pragma unroll
            for (int v = 0; v < NH; ++v) {
                const int i = (v * TPR + l) * VEC;
                x[v].forget();
                if (i < C) sum_of(x[v], i);
            }
            beyond(sum_of);
            if constexpr (W == 1) s = group_all<64, OpAdd>(s); else s = block_all<W, OpAdd>(s, sm, turn);
            const bool bad = q.label >= C;
            nll = bad ? __builtin_nanf("") : q.w * (logf(s) + (m - zl));
            if (dz) {
                const float g = bad ? __builtin_nanf("") : q.g, p = g / s;
                const int label = q.label;
                auto give = [&](const Packed<T> &x, int i) {
                    const int at = min(i, C - VEC), hit = label - at;
                    float o[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o[j] = exp_row<T>(x.get(j) - m) * p;
                    if (hit >= 0 && hit < VEC) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) o[j] -= j == hit ? g : 0.0f;
                    }
                    store_n<T, VEC>(dz + at, o);
                };
                beyond(give);
                // the next row's vectors come in as this row's go out
                enter(next);
                fetched = true;
#pragma unroll
                for (int v = 0; v < NH; ++v) {
                    const int i = (v * TPR + l) * VEC;
                    x[v].forget();
                    if (i < C) give(x[v], i);
                    if (q.label >= 0) fetch(v);
                }
            }
        } else if (dz) {
            const float o[VEC] = {};
            for (int i = l * VEC; i < C; i += TPR * VEC) store_n<T, VEC>(dz + min(i, C - VEC), o);
        }
        if (l == 0) {
            if (a.nll) a.nll[r] = nll;
            sum += (double)nll;
        }
        if (!fetched) {
            enter(next);
            if (q.label >= 0) {
#pragma unroll
                for (int v = 0; v < NH; ++v) fetch(v);
            }
        }
        r = next;
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
        a.n_wsum = (int)std::min<uint32_t>((a.s.rows + 4095) / 4096, LOSS_WSUM);
        hipLaunchKernelGGL(k_loss_weights, dim3(a.n_wsum), dim3(1024), 0, st, a, ws);
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
