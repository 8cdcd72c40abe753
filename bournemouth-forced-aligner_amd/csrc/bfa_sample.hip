// bfa_sample.hip -- one label per row of logits [B, T, C], drawn with temperature, top-k, top-p and min-p from a given number u.
//
//   m = max z;  x_i = (z_i - m) / T (0 where z_i = m);  w_i = exp(x_i);  NaN counts as -inf
//   order: z descending, index ascending.  Kept is the shortest of three prefixes, never empty: the first k; the shortest one
//   whose mass reaches p * mass(first k); the classes with w >= q
//   W = mass kept;  label = the lowest i with (kept mass up to and including i) > u W;  logp = x_label - log W
//
// Which side of a border between two classes u W falls on, and which class is the last one kept, are decisions: they are the
// same for every order of the work as long as the masses are good to far more digits than u has (24 bits).  They are made in
// float64, or in float32 where no border lies within the error of the sums (draw_fast); sums have a fixed order, no atomics on
// floats.
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

// y r + c with the constant in a pair of scalar registers (left to itself the compiler moves every constant of a polynomial into
// vector registers first, an instruction each).  The product itself is the compiler's: in inline asm it would not be kept apart from a
// v_readlane that has just brought a spilled constant back.
__device__ __forceinline__ double fma_c(double y, double r, double c)
{
    asm("" : "+s"(c));
    return __builtin_fma(y, r, c);
}
// e^x, x <= 0, to about one unit in the last place: x = n ln 2 + r, |r| <= ln 2 / 2, the Taylor polynomial of degree 12
// (remainder 0.3466^13 / 13! < 2^-52); -inf and NaN give 0.  The sum with 1.5 2^52 rounds to a whole number and holds it in its low
// bits.
__device__ __forceinline__ double exp_d(double x)
{
    const double big = 6755399441055744.0, sum = __builtin_fma(x, 1.4426950408889634, big), n = sum - big;
    double r = __builtin_fma(n, -0.69314718055994530942, x);  // ln 2 as a double (the product is not rounded) ...
    r = __builtin_fma(n, -2.3190468138462995584e-17, r);      // ... and what that lacks of ln 2
    double y = fma_c(r, 1.0 / 479001600.0, 1.0 / 39916800.0);
    y = fma_c(y, r, 1.0 / 3628800.0);
    y = fma_c(y, r, 1.0 / 362880.0);
    y = fma_c(y, r, 1.0 / 40320.0);
    y = fma_c(y, r, 1.0 / 5040.0);
    y = fma_c(y, r, 1.0 / 720.0);
    y = fma_c(y, r, 1.0 / 120.0);
    y = fma_c(y, r, 1.0 / 24.0);
    y = fma_c(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    y = __builtin_fma(y, r, 1.0);
    return x > -745.0 ? __builtin_ldexp(y, (int)(uint32_t)__double_as_longlong(sum)) : 0.0;
}
__device__ __forceinline__ double weight(float z, float m, double inv_t)
{
    return exp_d(z == m ? 0.0 : ((double)z - (double)m) * inv_t); // (both may be +inf)
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

// A row's draw in float32, by a group of G lanes of E consecutive classes each (z: -inf where a lane has none): false where a
// border lies within the error of the sums, so that the decision is left to float64.  In units of 2^-24, with A = log2 G steps over the lanes:
//   a weight 2^((z - m) log2(e) / T) carries three roundings of its exponent, |x| 3 w <= 1.11, and the exponential's 2 w: 1.11 C + 2 S
//   in any sum over the row;
//   a prefix up to a value adds E + A times, then once for a number of equal weights and once for their product at each of `steps`
//   values walked past, and twice at the last: 2 S + (E + A + 2 steps + 2) S;  p S: (E + A + 2 + 1) S;
//   the mass up to a class adds E times in the lanes in front, A over them, once more and E times in its own lane: (2 E + A + 1) S;
//   u W: (E + A + 1) S.
// So a prefix and p S differ by at most 2.22 C + (2 E + 2 A + 2 steps + 9) S more or less than they seem to, the mass up to a class
// and u W by 2.22 C + (3 E + 2 A + 6) S.  Only the label is certain in this way: logp is the float32 logarithm of W, off by
// (1.11 C / W + E + A + 2) 2^-24 and by the roundings of the logarithm itself.
template <int G, int E>
__device__ __forceinline__ bool draw_fast(const float (&z)[E], int at, int C, float m, const Draw &d, float u, int l, int &label, float &logp)
{
    const float NINF = -__builtin_inff();
    const float rate = (float)(d.inv_t * 1.4426950408889634);
    if (!(rate > 1e-20f && rate < 1e20f && fabsf(m) < 1e30f)) return false; // (the same for the lanes of a group)
    float w[E], S = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) { w[j] = __builtin_amdgcn_exp2f((z[j] - m) * rate); S += w[j]; }
    S = group_all<G, OpAdd>(S);
    constexpr float U = 1.0f / 16777216.0f, ADDS = 3 * E + (G == 4 ? 4 : G == 16 ? 8 : 12) + 10;
    const float tol = (2.25f * (float)C + ADDS * S) * U; // (U, ADDS: covers either bound without `steps`)
    float zt = NINF; // kept: z > zt, and of the classes at zt the first `ties`
    int ties = C;
    bool cut = false, sure = true;
    // (the median with +inf is the maximum; fmaxf would first quieten NaN, of which there are none)
    auto next_below = [&](float v) { // the greatest value under v
        float x = NINF;
#pragma unroll
        for (int j = 0; j < E; ++j) x = __builtin_amdgcn_fmed3f(x, z[j] < v ? z[j] : NINF, __builtin_inff());
        return group_all<G, OpMax>(x);
    };
    auto next_from = [&](float v) { // or at v
        float x = NINF;
#pragma unroll
        for (int j = 0; j < E; ++j) x = __builtin_amdgcn_fmed3f(x, z[j] <= v ? z[j] : NINF, __builtin_inff());
        return group_all<G, OpMax>(x);
    };
    auto count_at = [&](float v) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) c += z[j] == v ? 1 : 0;
        return group_all<G, OpAdd>(c);
    };
    auto mass_above = [&](float v) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) s += z[j] > v ? w[j] : 0.0f;
        return group_all<G, OpAdd>(s);
    };
    if (d.k < C) {
        float hi = m;
        int n = 0; // classes above hi
        if (d.k > 8) { // halve the range of the values a few times before walking down
            float lo = m;
#pragma unroll
            for (int j = 0; j < E; ++j) lo = z[j] > NINF ? fminf(lo, z[j]) : lo;
            lo = group_all<G, OpMin>(lo);
            for (int i = 0; i < 6; ++i) {
                const float mid = 0.5f * (lo + hi);
                int c = 0;
#pragma unroll
                for (int j = 0; j < E; ++j) c += z[j] > mid ? 1 : 0;
                c = group_all<G, OpAdd>(c);
                const bool below = c < d.k;
                n = below ? c : n;
                hi = below ? mid : hi;
                lo = below ? lo : mid;
            }
        }
        float v = next_from(hi);
        while (v > NINF) {
            const int c = count_at(v);
            if (n + c >= d.k) {
                zt = v;
                ties = d.k - n;
                cut = ties < c;
                break;
            }
            n += c;
            v = next_below(v);
        }
        if (zt > NINF && d.p < 1.0) S = mass_above(zt) + (float)ties * __builtin_amdgcn_exp2f((zt - m) * rate);
    }
    if (d.p < 1.0) {
        const float p = (float)d.p, target = p * S;
        float hi = m, M = 0.0f; // mass above hi
        // classes of weight (1 - p) S / C hold less than what is left out
        float lo = m + __builtin_amdgcn_logf((1.0f - p) * S / (float)C) / rate;
        for (int i = 0; i < 9; ++i) {
            const float mid = 0.5f * (lo + hi), s = mass_above(mid);
            const bool below = s < target;
            M = below ? s : M;
            hi = below ? mid : hi;
            lo = below ? lo : mid;
        }
        float v = next_from(hi), walked = tol;
        sure = false;
        while (v > NINF) {
            const int c = count_at(v);
            const float wv = __builtin_amdgcn_exp2f((v - m) * rate);
            if (!(M + (float)c * wv < target)) {
                const float r = fminf(fmaxf(ceilf((target - M) / wv), 1.0f), (float)c);
                zt = v;
                ties = (int)r;
                cut = ties < c;
                sure = target - (M + (r - 1.0f) * wv) > walked && (M + r * wv) - target > walked;
                break;
            }
            M += (float)c * wv;
            walked += 2.0f * U * S;
            v = next_below(v);
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) w[j] = z[j] >= zt ? w[j] : 0.0f;
    if (__any(cut)) {
        int before = 0; // classes at zt with a lower index
#pragma unroll
        for (int j = 0; j < E; ++j) before += (z[j] == zt) ? 1 : 0;
        before = group_scan<G>(before, l) - before;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool tie = z[j] == zt;
            w[j] = (tie & (before >= ties)) ? 0.0f : w[j];
            before += tie ? 1 : 0;
        }
    }
    const float q = (float)d.q;
    if (q > 0.0f) {
        bool near = false;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool top = z[j] == m;
            near |= !top & (w[j] > 0.0f) & (fabsf(w[j] - q) <= q * 3.0517578125e-5f); // (2^-15 > (3 |x| + 2) 2^-24 up to |x| = 170)
            w[j] = (top | (w[j] >= q)) ? w[j] : 0.0f;
        }
        sure = sure && !near;
    }
    float L = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) L += w[j];
    const float incl = group_scan<G>(L, l);
    const float W = __shfl(incl, G - 1, G), target = u * W;
    const int base = (threadIdx.x & 63) - l;
    const unsigned long long group = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1ull)) << base;
    const unsigned long long past = __ballot(incl > target) & group;
    if (!past) return false;
    const int lane = __ffsll((long long)past) - 1;
    // the class: as many as do not pass the target stand in front of it
    float run = incl - L, in_front = run, upto = __builtin_inff();
    int pick = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        run += w[j];
        const bool under = run <= target;
        pick += under ? 1 : 0;
        in_front = under ? run : in_front; // (run only grows)
        upto = __builtin_amdgcn_fmed3f(under ? __builtin_inff() : run, upto, -__builtin_inff());
    }
    float zp = z[0];
#pragma unroll
    for (int j = 1; j < E; ++j) zp = pick == j ? z[j] : zp;
    const bool good = (pick < E) & (upto - target > tol) & (target - in_front > tol);
    const unsigned long long ok = __ballot(good), bad = __ballot(!sure) & group;
    if (!((ok >> lane) & 1) || bad) return false;
    label = __shfl(at + pick, lane);
    zp = __shfl(zp, lane);
    logp = (float)(((double)zp - (double)m) * d.inv_t) - __builtin_amdgcn_logf(W) * 0.693147181f;
    return true;
}

// Short rows (C <= 512): G lanes share a row, each holds E consecutive classes.  Bound: instructions -- the draw in float32, with
// the end of a prefix bracketed by halving, and float64 for the rows that float32 leaves undecided (about one in a thousand).
// 4096 x 1000 rows of 67 float32 logits with top-p 0.73 ms (16 lanes to a row 1.27, everything in float64 and walking down from the
// top 4.6); 300 x 1500 ragged rows of 17 float16 logits with top-k 21 us (37).  The former take 1474 vector instructions per
// 16 rows: 0.61 ms at 4 cycles each.
template <typename T, int G, int E> __global__ __launch_bounds__(256) void k_sample_short(SampleArgs a)
{
    constexpr int RPG = 256 / G;
    const float NINF = -__builtin_inff();
    const int l = threadIdx.x % G, C = a.s.C;
    const int first = l * E, at = min(first, C - E);
    const int skip = first < C ? first - at : E; // the elements of a chunk moved back that are its neighbour's; all of one behind the row
    const bool each = a.p.temperature_B || a.p.top_p_B || a.p.min_p_B || a.p.top_k_B;
    Draw d = draw_of(a, 0);
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
                z[j] = j >= skip ? clean(z[j]) : NINF;
                m = fmaxf(m, z[j]);
            }
            m = group_all<G, OpMax>(m);
            if (each) d = draw_of(a, b);
            if (m > NINF && d.greedy) {
                int i = C;
#pragma unroll
                for (int j = E - 1; j >= 0; --j) i = (z[j] == m) ? at + j : i;
                label = group_all<G, OpMin>(i);
            } else if (m > NINF && !draw_fast<G, E>(z, at, C, m, d, a.u[r], l, label, logp)) {
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
// A prefix of the order is found without sorting the row:
//   k <= SAMPLE_LIST_K: at least k classes are no smaller than the k-th greatest of the 256 maxima of 4 threads each.  One sweep
//     collects the classes from there up (k = 50: about 56 of them), they are sorted, and the draw is made among them.
//   otherwise: a histogram of numbers and masses over 2048 ranges of the distance m - z shows the range the prefix ends in, one more
//     sweep collects that range and sorts it (a range of too many classes is divided by 2048 again).  Masses are whole multiples
//     of 2^-43 or finer there: integer atomics, whose order does not matter.
//   ranges that still hold too many (thousands of equal or extreme logits): the border is searched bit by bit, a sweep each.
// The draw itself adds the kept masses of blocks of 64 vectors in index order.
// Bound: the float64 exponentials of the histogram and of the draw where k does not bound the prefix, latency for few rows.  One
// workgroup per CU (with two, 64 registers a thread, the float64 polynomial spills: 604 us instead of 235 at the time).
// 512 rows of 131072 bfloat16 logits with parameters of their own 0.19 ms (searching every border bit by bit: 2.9), all with
// k = 50 63 us, all with p = 0.9 0.33 ms; 8 rows of 32000 float32 logits 43 us (472).
constexpr int SAMPLE_MAX_C = 1 << 19, SAMPLE_BLOCKS = SAMPLE_MAX_C / (64 * 4);
constexpr int SAMPLE_LIST = 2048, SAMPLE_LIST_K = 224, SAMPLE_BINS = 2048;

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
    // f(index, value) for every class, in vectors strided over the workgroup, U of them in flight
    template <int U, typename F> __device__ __forceinline__ void sweep(F &&f) const
    {
        const int n = C / VEC * VEC;
        int i = threadIdx.x * VEC;
        for (; U > 1 && i + (U - 1) * 1024 * VEC < n; i += U * 1024 * VEC) {
            float v[U][VEC];
#pragma unroll
            for (int k = 0; k < U; ++k) load_n<T, VEC>(z + i + k * 1024 * VEC, v[k]);
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) f(i + k * 1024 * VEC + j, v[k][j]);
        }
        for (; i < n; i += 1024 * VEC) {
            float v[VEC];
            load_n<T, VEC>(z + i, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f(i + j, v[j]);
        }
        if (n + (int)threadIdx.x < C) f(n + (int)threadIdx.x, (float)z[n + threadIdx.x]);
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

struct LongShared {
    union { unsigned long long bin[SAMPLE_BINS]; double mass[SAMPLE_BLOCKS]; };
    union { unsigned count[SAMPLE_BINS]; int tied[SAMPLE_BLOCKS]; };
    unsigned long long list[SAMPLE_LIST], sorted[SAMPLE_LIST]; // ~key << 32 | index: ascending is the order
    float top4[256];
    float f[32];
    double d[32];
    unsigned long long u[16];
    int i[32];
    int n;                    // length of the list
    uint32_t kt;              // where a prefix ends: its last key, how many classes of that key it holds ...
    int ties, all_ties;       // ... and how many there are
    double S;                 // the prefix's mass
    int at, front;            // the range it ends in, the number of classes in front of it
    unsigned long long front_mass, total;
};

template <typename T> struct LongSampler {
    using Row = LongRow<T>;
    LongShared &sh;
    const Row row;
    const float m;
    const double inv_t;
    int &tf, &td, &ti; // turns of block_all

    __device__ __forceinline__ unsigned long long entry(int i, float z) const { return ((unsigned long long)~key_of(z) << 32) | (unsigned)i; }
    __device__ __forceinline__ float entry_z(unsigned long long e) const { return value_of(~(uint32_t)(e >> 32)); }
    __device__ __forceinline__ double entry_w(unsigned long long e) const { return weight(entry_z(e), m, inv_t); }

    // the classes that `take` takes, sorted; -> their number, or more than SAMPLE_LIST (then nothing is sorted)
    template <typename F> __device__ __forceinline__ int collect(F &&take)
    {
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        row.template sweep<4>([&](int i, float z) {
            if (take(z)) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < SAMPLE_LIST) sh.list[at] = entry(i, z);
            }
        });
        __syncthreads();
        const int n = sh.n;
        if (n > SAMPLE_LIST) return n;
        for (int i = threadIdx.x; i < n; i += 1024) { // (each entry finds its place by itself: no steps to wait for each other)
            const unsigned long long e = sh.list[i];
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) place += sh.list[j] < e ? 1 : 0;
            sh.sorted[place] = e;
        }
        __syncthreads();
        return n;
    }

    __device__ __forceinline__ int count_from(uint32_t key)
    {
        int n = 0;
        row.template sweep<2>([&](int, float z) { n += key_of(clean(z)) >= key ? 1 : 0; });
        return block_all<16, OpAdd>(n, sh.i, ti);
    }
    __device__ __forceinline__ double mass_from(uint32_t key)
    {
        double M = 0.0;
        row.template sweep<1>([&](int, float z) { z = clean(z); if (key_of(z) >= key) M += weight(z, m, inv_t); });
        return block_all<16, OpAdd>(M, sh.d, td);
    }

    // where the first k classes (k > 0) or the shortest prefix of mass p S (k = 0; S < 0: of the whole row) end -> sh.kt, ties,
    // all_ties, S; k: at most the number of classes above -inf
    __device__ __forceinline__ void locate(int k, double p, double S)
    {
        const int shift = min(51, 31 + __clz(row.C)); // C 2^shift < 2^63
        const double up = __builtin_ldexp(1.0, shift), down = __builtin_ldexp(1.0, -shift);
        const float scale = (float)fmin((double)SAMPLE_BINS / 40.0 * inv_t, 1e37);
        float base = 0.0f, width = (float)SAMPLE_BINS, fine = 1.0f;
        int front = 0;
        unsigned long long front_mass = 0;
        double target = 0.0;
        auto place = [&](float z) { return fminf(z == m ? 0.0f : (m - z) * scale, (float)SAMPLE_BINS - 0.5f); }; // decreasing in z
        bool listed = false;
        int n = 0;
        for (int level = 0; level < 2 && !listed; ++level) {
            __syncthreads();
            for (int i = threadIdx.x; i < SAMPLE_BINS; i += 1024) { sh.bin[i] = 0; sh.count[i] = 0; }
            __syncthreads();
            row.template sweep<1>([&](int, float z) {
                const float v = place(z);
                // 2^52 + w 2^shift: its low bits are the whole number (not behind the branch: the vector's exponentials run side by side)
                const double x = __builtin_fma(weight(z, m, inv_t), up, 4503599627370496.0);
                if (z > -__builtin_inff() && v >= base && v < base + width) {
                    const int b = (int)((v - base) * fine);
                    atomicAdd(&sh.count[b], 1u);
                    atomicAdd(&sh.bin[b], (unsigned long long)__double_as_longlong(x) & 0xfffffffffffffull);
                }
            });
            __syncthreads();
            // two ranges per thread; prefix over the workgroup
            const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
            const int c0 = (int)sh.count[2 * t], c1 = (int)sh.count[2 * t + 1];
            const unsigned long long m0 = sh.bin[2 * t], m1 = sh.bin[2 * t + 1];
            int cs = group_scan<64>(c0 + c1, lane);
            unsigned long long ms = group_scan<64>(m0 + m1, lane);
            if (lane == 63) { sh.i[wave] = cs; sh.u[wave] = ms; }
            if (t == 0) sh.at = -1;
            __syncthreads();
            unsigned long long total = 0;
            for (int w = 0; w < 16; ++w) {
                if (w < wave) { cs += sh.i[w]; ms += sh.u[w]; }
                total += sh.u[w];
            }
            if (level == 0) target = p * (S < 0.0 ? (double)total * down : S);
            cs += front - c0 - c1; // what is in front of this thread's ranges
            ms += front_mass - m0 - m1;
            auto ends = [&](int c, unsigned long long M) { return k > 0 ? c >= k : (double)M * down >= target; };
            if (!ends(cs, ms) && ends(cs + c0 + c1, ms + m0 + m1)) {
                const bool second = !ends(cs + c0, ms + m0);
                sh.at = 2 * t + (second ? 1 : 0);
                sh.front = cs + (second ? c0 : 0);
                sh.front_mass = ms + (second ? m0 : 0);
            }
            __syncthreads();
            const int at = sh.at;
            if (at < 0) break; // (k: fewer classes than that; a target of 0)
            front = sh.front;
            front_mass = sh.front_mass;
            const unsigned here = sh.count[at];
            const bool open = level == 0 && at == SAMPLE_BINS - 1; // everything farther away
            base += (float)at / fine;
            width = 1.0f / fine;
            if (here <= SAMPLE_LIST) {
                n = collect([&](float z) { const float v = place(z); return z > -__builtin_inff() && v >= base && v < base + width; });
                listed = true;
            } else if (open) break;
            fine *= (float)SAMPLE_BINS;
        }
        const double M0 = (double)front_mass * down;
        if (listed) {
            if (threadIdx.x < 64) {
                const int lane = threadIdx.x;
                double run = M0, mass = M0;
                int K = 0;
                for (int i0 = 0; i0 < n; i0 += 64) {
                    const double w = i0 + lane < n ? entry_w(sh.sorted[i0 + lane]) : 0.0;
                    const double s = group_scan<64>(w, lane);
                    const unsigned long long in = __ballot(i0 + lane < n && (k > 0 ? front + i0 + lane < k : run + (s - w) < target));
                    if (in) { K = i0 + 64 - __clzll((long long)in); mass = run + __shfl(s, 63 - __clzll((long long)in)); }
                    run += __shfl(s, 63);
                }
                if (K < 1) K = 1; // (a target that rounding put in front of the range)
                const uint32_t key = (uint32_t)(sh.sorted[K - 1] >> 32);
                int ties = 0, all = 0;
                for (int i0 = 0; i0 < n; i0 += 64) {
                    const bool same = i0 + lane < n && (uint32_t)(sh.sorted[i0 + lane] >> 32) == key;
                    ties += __popcll(__ballot(same && i0 + lane < K));
                    all += __popcll(__ballot(same));
                }
                if (lane == 0) { sh.kt = ~key; sh.ties = ties; sh.all_ties = all; sh.S = mass; }
            }
            __syncthreads();
            return;
        }
        // bit by bit: the largest key with at least k classes, or the target's mass, from it up
        uint32_t key = 0;
        int ties, all;
        double mass;
        if (k > 0) {
            for (int bit = 31; bit >= 0; --bit)
                if (count_from(key | (1u << bit)) >= k) key |= 1u << bit;
            const int above = key == ~0u ? 0 : count_from(key + 1);
            all = count_from(key) - above;
            ties = k - above;
            mass = (key == ~0u ? 0.0 : mass_from(key + 1)) + (double)ties * weight(value_of(key), m, inv_t);
        } else {
            for (int bit = 31; bit >= 0; --bit)
                if (mass_from(key | (1u << bit)) >= target) key |= 1u << bit;
            const double M = key == ~0u ? 0.0 : mass_from(key + 1);
            all = count_from(key) - (key == ~0u ? 0 : count_from(key + 1));
            ties = max(ties_taken(M, weight(value_of(key), m, inv_t), all, target), 1);
            mass = M;
        }
        __syncthreads();
        if (threadIdx.x == 0) { sh.kt = key; sh.ties = ties; sh.all_ties = all; sh.S = mass; }
        __syncthreads();
    }

    // the draw among the first k of the n sorted classes (one wave, at most 4 each)
    __device__ __forceinline__ void draw_listed(int n, const Draw &d, float u, int32_t *label, float *logp)
    {
        constexpr int E = (SAMPLE_LIST_K + 63) / 64;
        const int lane = threadIdx.x, kk = min(n, d.k);
        unsigned long long e[E];
        double w[E], in_front[E], S = 0.0;
#pragma unroll
        for (int c = 0; c < E; ++c) {
            const int i = c * 64 + lane;
            e[c] = i < kk ? sh.sorted[i] : ~0ull;
            w[c] = i < kk ? entry_w(e[c]) : 0.0;
            const double s = group_scan<64>(w[c], lane);
            in_front[c] = S + (s - w[c]);
            S += __shfl(s, 63);
        }
        const double target = d.p * S;
#pragma unroll
        for (int c = 0; c < E; ++c)
            if (!(w[c] >= d.q) || (d.p < 1.0 && !(in_front[c] < target))) w[c] = 0.0;
        double upto[E] = {}, W = 0.0; // the kept mass up to a class and in all, added in the same order
#pragma unroll
        for (int c = 0; c < E; ++c) {
            unsigned long long some = __ballot(w[c] > 0.0);
            while (some) {
                const int from = __ffsll((long long)some) - 1;
                some &= some - 1;
                const double wj = __shfl(w[c], from);
                const uint32_t ij = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)e[c], from);
                W += wj;
#pragma unroll
                for (int q = 0; q < E; ++q) upto[q] += ij <= (uint32_t)e[q] ? wj : 0.0;
            }
        }
        const double goal = target_of(u, W);
        int first = 0x7fffffff, last = -1;
#pragma unroll
        for (int c = 0; c < E; ++c)
            if (w[c] > 0.0) {
                const int i = (int)(uint32_t)e[c];
                if (upto[c] > goal) first = min(first, i);
                last = max(last, i);
            }
        first = group_all<64, OpMin>(first);
        last = group_all<64, OpMax>(last);
        const int pick = first != 0x7fffffff ? first : last;
#pragma unroll
        for (int c = 0; c < E; ++c)
            if (w[c] > 0.0 && (int)(uint32_t)e[c] == pick) {
                *label = pick;
                if (logp) *logp = logp_of(entry_z(e[c]), m, inv_t, W);
            }
    }
};

template <typename T> __global__ __launch_bounds__(1024, 4) void k_sample_long(SampleArgs a)
{
    using Row = LongRow<T>;
    constexpr int VEC = Row::VEC, W16 = 16;
    __shared__ LongShared sh;
    const float NINF = -__builtin_inff();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tf = 0, td = 0, ti = 0;
    for (uint32_t r = blockIdx.x; r < a.s.rows; r += gridDim.x) {
        uint32_t b, t;
        a.s.split(r, b, t);
        float mine = NINF, m = NINF;
        const Row row = {row_in<T>(a.z, b, t), a.s.C};
        __syncthreads(); // the shared memory is free again
        if (a.s.held(b, t)) {
            row.template sweep<4>([&](int, float z) { mine = fmaxf(mine, z); }); // (fmaxf passes over NaN)
            m = block_all<W16, OpMax>(mine, sh.f, tf);
        }
        if (m == NINF) { // (the same for all threads)
            if (threadIdx.x == 0) { a.label[r] = -1; if (a.logp) a.logp[r] = 0.0f; }
            continue;
        }
        const Draw d = draw_of(a, b);
        if (d.greedy) {
            int i = a.s.C;
            row.template sweep<4>([&](int j, float z) { i = z == m ? min(i, j) : i; });
            i = block_all<W16, OpMin>(i, sh.i, ti);
            if (threadIdx.x == 0) { a.label[r] = i; if (a.logp) a.logp[r] = 0.0f; }
            continue;
        }
        LongSampler<T> own = {sh, row, m, d.inv_t, tf, td, ti};
        if (d.k <= SAMPLE_LIST_K) {
            const float q = group_all<4, OpMax>(mine);
            if ((lane & 3) == 0) sh.top4[threadIdx.x >> 2] = q;
            __syncthreads();
            if (wave == 0) { // the k-th greatest of the 256, bit by bit
                uint32_t key[4], kt = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c) key[c] = key_of(sh.top4[c * 64 + lane]);
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t x = kt | (1u << bit);
                    int n = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) n += __popcll(__ballot(key[c] >= x));
                    if (n >= d.k) kt = x;
                }
                if (lane == 0) sh.kt = kt;
            }
            __syncthreads();
            const float from = value_of(sh.kt); // (-inf where fewer groups hold anything)
            const int n = own.collect([&](float z) { return z >= from && z > NINF; });
            if (n <= SAMPLE_LIST) {
                if (wave == 0) own.draw_listed(n, d, a.u[r], a.label + r, a.logp ? a.logp + r : nullptr);
                continue;
            }
        }
        float zt = NINF; // kept: z > zt, and of the classes at zt the first `ties`
        int ties = a.s.C, all_ties = 0;
        double S = -1.0;
        if (d.k < a.s.C) {
            int n = 0;
            row.template sweep<4>([&](int, float z) { n += z > NINF ? 1 : 0; });
            n = block_all<W16, OpAdd>(n, sh.i, ti);
            if (d.k < n) {
                own.locate(d.k, 0.0, 0.0);
                zt = value_of(sh.kt); ties = sh.ties; all_ties = sh.all_ties; S = sh.S;
            }
        }
        if (d.p < 1.0) {
            own.locate(0, d.p, S);
            zt = value_of(sh.kt); ties = sh.ties; all_ties = sh.all_ties;
        }
        // of classes at zt those in front of every block of BLOCK classes, where not all of them are kept
        const int nb = (a.s.C + Row::BLOCK - 1) / Row::BLOCK;
        const bool cut = ties < all_ties;
        __syncthreads();
        if (cut) {
            for (int k = wave; k < nb; k += W16) {
                float z[VEC];
                int c = 0;
                row.block(k, z);
#pragma unroll
                for (int j = 0; j < VEC; ++j) c += z[j] == zt ? 1 : 0;
                c = group_all<64, OpAdd>(c);
                if (lane == 0) sh.tied[k] = c;
            }
            __syncthreads();
            if (wave == 0) { // exclusive prefix
                int run = 0;
                for (int k0 = 0; k0 < nb; k0 += 64) {
                    const int c = k0 + lane < nb ? sh.tied[k0 + lane] : 0;
                    const int s = group_scan<64>(c, lane);
                    if (k0 + lane < nb) sh.tied[k0 + lane] = run + s - c;
                    run += __shfl(s, 63);
                }
            }
            __syncthreads();
        }
        // the kept mass of every block, in index order
        auto kept = [&](int k, const float (&z)[VEC], double (&w)[VEC]) {
            int before = 0;
            if (cut) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) before += z[j] == zt ? 1 : 0;
                before = sh.tied[k] + group_scan<64>(before, lane) - before;
            }
            double L = 0.0;
            bool some = false;
#pragma unroll
            for (int j = 0; j < VEC; ++j) { some |= z[j] >= zt; w[j] = 0.0; }
            if (!__any(some)) return L;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                bool keep = z[j] >= zt;
                if (cut) {
                    const bool tie = z[j] == zt;
                    keep &= !tie | (before < ties);
                    before += tie ? 1 : 0;
                }
                const double x = weight(z[j], m, d.inv_t);
                w[j] = (keep & (x >= d.q)) ? x : 0.0;
                L += w[j];
            }
            return L;
        };
        for (int k = wave; k < nb; k += W16) {
            float z[VEC];
            double w[VEC];
            row.block(k, z);
            const double L = group_all<64, OpAdd>(kept(k, z, w));
            if (lane == 0) sh.mass[k] = L;
        }
        __syncthreads();
        if (wave == 0) {
            double W = 0.0;
            for (int k0 = 0; k0 < nb; k0 += 64) {
                const double s = group_scan<64>(k0 + lane < nb ? sh.mass[k0 + lane] : 0.0, lane);
                W += __shfl(s, 63);
            }
            const double target = target_of(a.u[r], W);
            // the block: the first whose mass passes the target, else the last with a weight
            double run = 0.0, before = 0.0, last_before = 0.0;
            int pick = -1, last = 0;
            for (int k0 = 0; k0 < nb && pick < 0; k0 += 64) {
                const double x = k0 + lane < nb ? sh.mass[k0 + lane] : 0.0;
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
            row.block(pick, z);
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
    }
}

template <typename T, int G, int E> static void sample_short(const SampleArgs &a, hipStream_t st)
{
    const uint32_t grid = std::min<uint32_t>((a.s.rows + 256 / G - 1) / (256 / G), 8192);
    hipLaunchKernelGGL((k_sample_short<T, G, E>), dim3(grid), dim3(256), 0, st, a);
}
// the fewest lanes a row fits in with at most 20 classes each: reductions over lanes serve more rows at a time
template <typename T, int G> static void sample_short_e(const SampleArgs &a, hipStream_t st)
{
    const int e = (a.s.C + G - 1) / G;
    if constexpr (G == 4) {
        if (e <= 1) return sample_short<T, G, 1>(a, st);
        if (e <= 2) return sample_short<T, G, 2>(a, st);
        if (e <= 3) return sample_short<T, G, 3>(a, st);
        if (e <= 4) return sample_short<T, G, 4>(a, st);
        if (e <= 5) return sample_short<T, G, 5>(a, st);
    }
    if (e <= 6) return sample_short<T, G, 6>(a, st);
    if (e <= 7) return sample_short<T, G, 7>(a, st);
    if constexpr (G == 64) return sample_short<T, G, 8>(a, st);
    else {
        if (e <= 8) return sample_short<T, G, 8>(a, st);
        if (e <= 10) return sample_short<T, G, 10>(a, st);
        if (e <= 12) return sample_short<T, G, 12>(a, st);
        if (e <= 14) return sample_short<T, G, 14>(a, st);
        if (e <= 17) return sample_short<T, G, 17>(a, st);
        return sample_short<T, G, 20>(a, st);
    }
}
template <typename T> static void sample_launch(const SampleArgs &a, hipStream_t st)
{
    if (a.s.C <= 80) sample_short_e<T, 4>(a, st);
    else if (a.s.C <= 320) sample_short_e<T, 16>(a, st);
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
