// bfa_sample.hip -- one label per row of logits [B, T, C], drawn with temperature, top-k, top-p and min-p from a given number u.
//
//   m = max z;  x_i = (z_i - m) / T (0 where z_i = m);  w_i = exp(x_i);  NaN counts as -inf
//   order: z descending, index ascending.  Kept is the shortest of three prefixes, never empty: the first k; the shortest one
//   whose mass reaches p * mass(first k); the classes with w >= q
//   W = mass kept;  label = the lowest i with (kept mass up to and including i) > u W;  logp = x_label - log W
//
// Which side of a border between two classes u W falls on, and which class is the last one kept, are decisions: they are the
// same for every order of the work as long as the masses are good to far more digits than u has (24 bits).  Weights and masses
// are therefore float64 (a float64 fma issues at the rate of a float32 one here); sums have a fixed order, no atomics.
#include <algorithm>

#include "bfa_rows.hpp"

namespace bfa {

struct SampleArgs {
    RowShape s;
    RowPtr z;
    const float *u;
    bfa_sample_params p;
    int32_t *label;
    float *logp; // or null
};

// the parameters of an utterance, resolved
struct Draw {
    double inv_t, p, q;
    int k;       // <= C
    bool greedy; // the first class of the order alone
};
__device__ __forceinline__ Draw draw_of(const SampleArgs &a, uint32_t b)
{
    const float t = a.p.temperature_B ? a.p.temperature_B[b] : a.p.temperature;
    const float p = a.p.top_p_B ? a.p.top_p_B[b] : a.p.top_p;
    const float q = a.p.min_p_B ? a.p.min_p_B[b] : a.p.min_p;
    const int k = a.p.top_k_B ? a.p.top_k_B[b] : a.p.top_k;
    Draw d;
    d.greedy = !(t > 0.0f) || !(p > 0.0f) || !(q <= 1.0f); // (NaN too)
    d.inv_t = 1.0 / (double)t;
    d.p = (double)p;
    d.q = (double)q;
    d.k = (k <= 0 || k > a.s.C) ? a.s.C : k;
    return d;
}

// e^x, x <= 0, to about one unit in the last place: x = n ln 2 + r, |r| <= ln 2 / 2, the Taylor polynomial of degree 12
// (remainder 0.3466^13 / 13! < 2^-52)
__device__ __forceinline__ double exp_d(double x)
{
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0.69314718055994530942, x);  // ln 2 as a double (the product is not rounded) ...
    r = __builtin_fma(n, -2.3190468138462995584e-17, r);      // ... and what that lacks of ln 2
    double y = 1.0 / 479001600.0;
    y = __builtin_fma(y, r, 1.0 / 39916800.0);
    y = __builtin_fma(y, r, 1.0 / 3628800.0);
    y = __builtin_fma(y, r, 1.0 / 362880.0);
    y = __builtin_fma(y, r, 1.0 / 40320.0);
    y = __builtin_fma(y, r, 1.0 / 5040.0);
    y = __builtin_fma(y, r, 1.0 / 720.0);
    y = __builtin_fma(y, r, 1.0 / 120.0);
    y = __builtin_fma(y, r, 1.0 / 24.0);
    y = __builtin_fma(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    y = __builtin_fma(y, r, 1.0);
    return x > -745.0 ? __builtin_ldexp(y, (int)n) : 0.0; // (-inf too)
}
__device__ __forceinline__ double weight(float z, float m, double inv_t)
{
    if (z == m) return 1.0;
    return z == -__builtin_inff() ? 0.0 : exp_d(((double)z - (double)m) * inv_t);
}
__device__ __forceinline__ float clean(float z) { return z == z ? z : -__builtin_inff(); }
__device__ __forceinline__ double target_of(float u, double W) { const double t = (double)u * W; return t > 0.0 ? t : 0.0; }
__device__ __forceinline__ float logp_of(float z, float m, double inv_t, double W)
{
    const double x = (z == m) ? 0.0 : ((double)z - (double)m) * inv_t;
    return (float)(x - (double)log1pf((float)(W - 1.0))); // W >= 1: its first class has weight 1
}
// of c classes of weight w each behind mass M: how many the prefix takes that stops when the mass in front reaches `target`
__device__ __forceinline__ int ties_taken(double M, double w, int c, double target)
{
    int r = (int)fmin(fmax(__builtin_ceil((target - M) / w), 0.0), (double)c);
    while (r > 0 && !(M + (double)(r - 1) * w < target)) --r;
    while (r < c && M + (double)r * w < target) ++r;
    return r;
}

// inclusive prefix over the G lanes of a group
template <int G, typename V> __device__ __forceinline__ V group_scan(V x, int l)
{
    if constexpr (G == 4) {
        V y = dpp<DPP_SHR + 1>(x); if (l >= 1) x += y;
        y = dpp<DPP_SHR + 2>(x); if (l >= 2) x += y;
    } else {
        const int q = l & 15;
        V y = dpp<DPP_SHR + 1>(x); if (q >= 1) x += y;
        y = dpp<DPP_SHR + 2>(x); if (q >= 2) x += y;
        y = dpp<DPP_SHR + 4>(x); if (q >= 4) x += y;
        y = dpp<DPP_SHR + 8>(x); if (q >= 8) x += y;
        if constexpr (G == 64) {
            y = __shfl(x, (l & 48) - 1); if (l & 16) x += y; // the row of 16 before, where this is the second of a pair
            y = __shfl(x, 31); if (l & 32) x += y;
        }
    }
    return x;
}

// Short rows (C <= 512): G lanes share a row, each holds E consecutive classes.  Bound: the float64 exponentials and, with top-k
// or top-p, the walk down the distinct values from the top (one maximum over the group per value).
template <typename T, int G, int E> __global__ __launch_bounds__(256) void k_sample_short(SampleArgs a)
{
    constexpr int RPG = 256 / G;
    const float NINF = -__builtin_inff();
    const int l = threadIdx.x % G, C = a.s.C;
    const int first = l * E, at = min(first, C - E);
    const bool on = first < C;
    for (uint32_t r = blockIdx.x * RPG + threadIdx.x / G; r < a.s.rows; r += gridDim.x * RPG) {
        uint32_t b, t;
        a.s.split(r, b, t);
        int label = -1;
        float logp = 0.0f;
        if (a.s.held(b, t)) { // (the same for the G lanes of a row)
            float z[E], m = NINF;
            load_n<T, E>(row_in<T>(a.z, b, t) + at, z);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                z[j] = (on && at + j >= first) ? clean(z[j]) : NINF;
                m = fmaxf(m, z[j]);
            }
            m = group_all<G, OpMax>(m);
            const Draw d = draw_of(a, b);
            if (m > NINF && d.greedy) {
                int i = C;
#pragma unroll
                for (int j = E - 1; j >= 0; --j) i = (z[j] == m) ? at + j : i;
                label = group_all<G, OpMin>(i);
            } else if (m > NINF) {
                double w[E], S = 0.0;
#pragma unroll
                for (int j = 0; j < E; ++j) { w[j] = weight(z[j], m, d.inv_t); S += w[j]; }
                float zt = NINF; // kept: z > zt, and of the classes at zt the first `ties`
                int ties = C;
                // down the distinct values until `done(number, mass so far, number at this value, weight)`
                auto walk = [&](auto &&done) {
                    float cur = __builtin_inff();
                    bool top = true;
                    int n = 0;
                    double M = 0.0;
                    for (;;) {
                        float v = NINF;
#pragma unroll
                        for (int j = 0; j < E; ++j) v = (z[j] < cur || top) ? fmaxf(v, z[j]) : v;
                        v = group_all<G, OpMax>(v);
                        if (v == NINF) return; // what is left weighs nothing
                        int c = 0;
#pragma unroll
                        for (int j = 0; j < E; ++j) c += (z[j] == v) ? 1 : 0;
                        c = group_all<G, OpAdd>(c);
                        const double wv = weight(v, m, d.inv_t);
                        if (done(n, M, c, wv)) { zt = v; return; }
                        n += c;
                        M += (double)c * wv;
                        cur = v;
                        top = false;
                    }
                };
                if (d.k < C || d.p < 1.0) S = group_all<G, OpAdd>(S);
                if (d.k < C)
                    walk([&](int n, double M, int c, double wv) {
                        if (n + c < d.k) return false;
                        ties = d.k - n;
                        S = M + (double)ties * wv;
                        return true;
                    });
                if (d.p < 1.0) {
                    const double target = d.p * S;
                    walk([&](int n, double M, int c, double wv) {
                        if (M + (double)c * wv < target) return false;
                        ties = max(ties_taken(M, wv, c, target), n == 0 ? 1 : 0);
                        return true;
                    });
                }
                int before = 0; // classes at zt with a lower index
#pragma unroll
                for (int j = 0; j < E; ++j) before += (z[j] == zt) ? 1 : 0;
                before = group_scan<G>(before, l) - before;
                double L = 0.0;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    bool keep = z[j] > zt;
                    if (z[j] == zt) { keep = before < ties; ++before; }
                    if (!(keep && w[j] >= d.q)) w[j] = 0.0;
                    L += w[j];
                }
                const double incl = group_scan<G>(L, l);
                const double W = __shfl(incl, G - 1, G);
                const double target = target_of(a.u[r], W);
                // the lane: the first whose mass passes the target, else (u >= 1) the last with a weight
                const int base = (threadIdx.x & 63) - l;
                const unsigned long long group = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1ull)) << base;
                const unsigned long long past = __ballot(incl > target && L > 0.0) & group, some = __ballot(L > 0.0) & group;
                const int lane = past ? __ffsll((long long)past) - 1 : 63 - __clzll((long long)some);
                // its class, likewise
                double run = incl - L;
                int pick = 0;
                bool found = false;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    run += w[j];
                    if (!found && w[j] > 0.0) { pick = j; found = past != 0ull && run > target; }
                }
                float zp = z[0];
#pragma unroll
                for (int j = 1; j < E; ++j) zp = (pick == j) ? z[j] : zp;
                label = __shfl(at + pick, lane);
                logp = logp_of(__shfl(zp, lane), m, d.inv_t, W);
            }
        }
        if (l == 0) {
            a.label[r] = label;
            if (a.logp) a.logp[r] = logp;
        }
    }
}

// ---- long rows: a workgroup of 1024 threads per row -------------------------------------------------------------------------
constexpr int SAMPLE_MAX_C = 1 << 19, SAMPLE_BLOCKS = SAMPLE_MAX_C / (64 * 4);

// float order as unsigned order (-0 as +0)
__device__ __forceinline__ uint32_t key_of(float z)
{
    const uint32_t u = __float_as_uint(z == 0.0f ? 0.0f : z);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

template <typename T> struct LongRow {
    static constexpr int VEC = 16 / sizeof(T), BLOCK = 64 * VEC;
    const T *z;
    int C;
    // f(index, value) for every class, in vectors strided over the workgroup
    template <typename F> __device__ __forceinline__ void sweep(F &&f) const
    {
        const int n = C / VEC * VEC;
        for (int i = threadIdx.x * VEC; i < n; i += 1024 * VEC) {
            float v[VEC];
            load_n<T, VEC>(z + i, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f(i + j, clean(v[j]));
        }
        if (n + (int)threadIdx.x < C) f(n + (int)threadIdx.x, clean((float)z[n + threadIdx.x]));
    }
    // this lane's VEC consecutive classes of block k (BLOCK classes, one wave); -inf behind the row
    __device__ __forceinline__ void block(int k, float (&v)[VEC]) const
    {
        const int i = k * BLOCK + (int)(threadIdx.x & 63) * VEC;
        if (i + VEC <= C) load_n<T, VEC>(z + i, v);
        else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = i + j < C ? (float)z[i + j] : -__builtin_inff();
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = clean(v[j]);
    }
};

template <typename T> __global__ __launch_bounds__(1024) void k_sample_long(SampleArgs a)
{
    using Row = LongRow<T>;
    constexpr int VEC = Row::VEC, W16 = 16;
    __shared__ float smf[2 * W16];
    __shared__ double smd[2 * W16];
    __shared__ int smi[2 * W16];
    __shared__ double mass[SAMPLE_BLOCKS];
    __shared__ int tied[SAMPLE_BLOCKS];
    const float NINF = -__builtin_inff();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tf = 0, td = 0, ti = 0;
    for (uint32_t r = blockIdx.x; r < a.s.rows; r += gridDim.x) {
        uint32_t b, t;
        a.s.split(r, b, t);
        float m = NINF;
        const Row row = {row_in<T>(a.z, b, t), a.s.C};
        if (a.s.held(b, t)) {
            row.sweep([&](int, float z) { m = fmaxf(m, z); });
            m = block_all<W16, OpMax>(m, smf, tf);
        }
        if (m == NINF) { // (the same for all threads)
            if (threadIdx.x == 0) { a.label[r] = -1; if (a.logp) a.logp[r] = 0.0f; }
            continue;
        }
        const Draw d = draw_of(a, b);
        if (d.greedy) {
            int i = a.s.C;
            row.sweep([&](int j, float z) { if (z == m) i = min(i, j); });
            i = block_all<W16, OpMin>(i, smi, ti);
            if (threadIdx.x == 0) { a.label[r] = i; if (a.logp) a.logp[r] = 0.0f; }
            continue;
        }
        uint32_t kt = 0; // kept: key > kt, and of the classes at kt the first `ties`
        int ties = a.s.C;
        auto count_from = [&](uint32_t key) {
            int n = 0;
            row.sweep([&](int, float z) { n += key_of(z) >= key ? 1 : 0; });
            return block_all<W16, OpAdd>(n, smi, ti);
        };
        auto mass_from = [&](uint32_t key) {
            double M = 0.0;
            row.sweep([&](int, float z) { if (key_of(z) >= key) M += weight(z, m, d.inv_t); });
            return block_all<W16, OpAdd>(M, smd, td);
        };
        double S = 0.0;
        if (d.k < a.s.C) { // the largest key with at least k classes from it up, bit by bit
            for (int bit = 31; bit >= 0; --bit)
                if (count_from(kt | (1u << bit)) >= d.k) kt |= 1u << bit;
            ties = d.k - (kt == ~0u ? 0 : count_from(kt + 1));
            S = (kt == ~0u ? 0.0 : mass_from(kt + 1)) + (double)ties * weight(value_of(kt), m, d.inv_t);
        } else if (d.p < 1.0) S = mass_from(0);
        if (d.p < 1.0) { // the largest key with at least the target's mass from it up
            const double target = d.p * S;
            uint32_t kp = 0;
            for (int bit = 31; bit >= 0; --bit)
                if (mass_from(kp | (1u << bit)) >= target) kp |= 1u << bit;
            const double M = kp == ~0u ? 0.0 : mass_from(kp + 1);
            const int c = count_from(kp) - (kp == ~0u ? 0 : count_from(kp + 1));
            kt = kp;
            ties = max(ties_taken(M, weight(value_of(kp), m, d.inv_t), c, target), 1);
        }
        // the kept mass of every block of BLOCK classes, in index order
        const int nb = (a.s.C + Row::BLOCK - 1) / Row::BLOCK;
        __syncthreads();
        for (int k = wave; k < nb; k += W16) {
            float z[VEC];
            int c = 0;
            row.block(k, z);
#pragma unroll
            for (int j = 0; j < VEC; ++j) c += key_of(z[j]) == kt ? 1 : 0;
            c = group_all<64, OpAdd>(c);
            if (lane == 0) tied[k] = c;
        }
        __syncthreads();
        if (wave == 0) { // exclusive prefix
            int run = 0;
            for (int k0 = 0; k0 < nb; k0 += 64) {
                const int c = k0 + lane < nb ? tied[k0 + lane] : 0;
                const int s = group_scan<64>(c, lane);
                if (k0 + lane < nb) tied[k0 + lane] = run + s - c;
                run += __shfl(s, 63);
            }
        }
        __syncthreads();
        auto kept = [&](int k, float (&z)[VEC], double (&w)[VEC]) {
            row.block(k, z);
            int before = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) before += key_of(z[j]) == kt ? 1 : 0;
            before = tied[k] + group_scan<64>(before, lane) - before;
            double L = 0.0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t key = key_of(z[j]);
                bool keep = key > kt;
                if (key == kt) { keep = before < ties; ++before; }
                w[j] = keep ? weight(z[j], m, d.inv_t) : 0.0;
                if (!(w[j] >= d.q)) w[j] = 0.0;
                L += w[j];
            }
            return L;
        };
        for (int k = wave; k < nb; k += W16) {
            float z[VEC];
            double w[VEC];
            const double L = group_all<64, OpAdd>(kept(k, z, w));
            if (lane == 0) mass[k] = L;
        }
        __syncthreads();
        if (wave == 0) {
            double W = 0.0;
            for (int k0 = 0; k0 < nb; k0 += 64) {
                const double s = group_scan<64>(k0 + lane < nb ? mass[k0 + lane] : 0.0, lane);
                W += __shfl(s, 63);
            }
            const double target = target_of(a.u[r], W);
            // the block: the first whose mass passes the target, else the last with a weight
            double run = 0.0, before = 0.0, last_before = 0.0;
            int pick = -1, last = 0;
            for (int k0 = 0; k0 < nb && pick < 0; k0 += 64) {
                const double x = k0 + lane < nb ? mass[k0 + lane] : 0.0;
                const double s = group_scan<64>(x, lane);
                const unsigned long long past = __ballot(run + s > target && x > 0.0), some = __ballot(x > 0.0);
                const int at = past ? __ffsll((long long)past) - 1 : (some ? 63 - __clzll((long long)some) : 0);
                const double front = run + __shfl(s - x, at);
                if (past) { pick = k0 + at; before = front; }
                else if (some) { last = k0 + at; last_before = front; }
                run += __shfl(s, 63);
            }
            const bool any = pick >= 0;
            if (!any) { pick = last; before = last_before; }
            float z[VEC];
            double w[VEC];
            const double L = kept(pick, z, w);
            const double incl = group_scan<64>(L, lane) + before;
            const unsigned long long past = any ? __ballot(incl > target && L > 0.0) : 0ull, some = __ballot(L > 0.0);
            const int at = past ? __ffsll((long long)past) - 1 : 63 - __clzll((long long)some);
            double go = incl - L;
            int j0 = 0;
            bool found = false;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                go += w[j];
                if (!found && w[j] > 0.0) { j0 = j; found = past != 0ull && go > target; }
            }
            float zp = z[0];
#pragma unroll
            for (int j = 1; j < VEC; ++j) zp = (j0 == j) ? z[j] : zp;
            if (lane == at) {
                a.label[r] = pick * Row::BLOCK + lane * VEC + j0;
                if (a.logp) a.logp[r] = logp_of(zp, m, d.inv_t, W);
            }
        }
        __syncthreads(); // mass and tied are free again
    }
}

template <typename T, int G, int E> static void sample_short(const SampleArgs &a, hipStream_t st)
{
    const uint32_t grid = std::min<uint32_t>((a.s.rows + 256 / G - 1) / (256 / G), 8192);
    hipLaunchKernelGGL((k_sample_short<T, G, E>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T, int G> static void sample_short_e(const SampleArgs &a, hipStream_t st)
{
    switch ((a.s.C + G - 1) / G) {
    case 1: return sample_short<T, G, 1>(a, st);
    case 2: return sample_short<T, G, 2>(a, st);
    case 3: return sample_short<T, G, 3>(a, st);
    case 4: return sample_short<T, G, 4>(a, st);
    case 5: return sample_short<T, G, 5>(a, st);
    case 6: return sample_short<T, G, 6>(a, st);
    case 7: return sample_short<T, G, 7>(a, st);
    default: return sample_short<T, G, 8>(a, st);
    }
}
template <typename T> static void sample_launch(const SampleArgs &a, hipStream_t st)
{
    if (a.s.C <= 32) sample_short_e<T, 4>(a, st);
    else if (a.s.C <= 128) sample_short_e<T, 16>(a, st);
    else if (a.s.C <= 512) sample_short_e<T, 64>(a, st);
    else hipLaunchKernelGGL((k_sample_long<T>), dim3(std::min<uint32_t>(a.s.rows, 1024)), dim3(1024), 0, st, a);
}

} // namespace bfa

extern "C" int bfa_sample_max_c() { return bfa::SAMPLE_MAX_C; }

extern "C" int bfa_launch_sample(const bfa_rows *z, int B, int T, int C, const int32_t *T_len, const float *u, const bfa_sample_params *p,
                                 int32_t *label, float *logp, void *stream)
{
    using namespace bfa;
    const SampleArgs a{RowShape(B, T, C, T_len), {z->data, z->strideB, z->strideT}, u, *p, label, logp};
    if (z->dtype == BFA_F32) sample_launch<float>(a, (hipStream_t)stream);
    else if (z->dtype == BFA_F16) sample_launch<_Float16>(a, (hipStream_t)stream);
    else sample_launch<__bf16>(a, (hipStream_t)stream);
    return (int)hipGetLastError();
}
