// Draw of one index per row of logits, with temperature, top-k, top-p and min-p, from given uniform numbers:
//     z_i = l_i / temperature,  w_i = exp(z_i - max z);  order: larger logit first, equal ones by index
//     top-k   the first k of the order             top-p   of those, the shortest prefix whose mass reaches p of theirs
//     min-p   w_i >= min_p (of the largest)        draw    in index order, the first i with w_0 + .. + w_i > u * sum
// The kept set is always a prefix of the order, so it is described by its last element (value, index).  Weights are
// held as 64-bit integers, w 2^43 rounded: their sums do not depend on the order of adding, so LDS atomics and any
// launch shape give the same index, and a row of 2^20 logits cannot overflow.  exp is evaluated in float64: an index
// depends on which side of a border a sum of many weights falls.
// NaN counts as -inf; +inf takes all the mass (several share it); a row without a finite or +inf logit gives index -1
// and log-probability -inf.  temperature <= 0: the first largest logit.
// Rows of up to 64 logits: a group of lanes per row, everything in registers.  Longer rows: a workgroup per row, which
// reads its row a few times (the first time from HBM, then from L2): maximum; counts and masses over 2048 bins of
// 1/64 nat below the maximum; the elements of the bin in which a border falls, sorted in LDS; the masses of the kept.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "marl_env.h"
#include "marl_net.h"
#include "marl_types.h"

extern "C" __attribute__((visibility("hidden"))) void marl_note_hip_error(int err);     // marl_env.hip

namespace {

using namespace marl_types;
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int64_t ld, rows;
    int32_t V;
    const float* u;
    const float* settings;          // [rows][4] or NULL
    float temperature, top_p, min_p;
    int32_t top_k;
    int64_t* index;
    float* log_prob;
};

struct Rule {                       // one row's settings, made safe
    double inv_t, p, log_m;         // p >= 1: off;  log_m = -inf: off
    int32_t k;                      // 0: off
    bool greedy;
};

__device__ __forceinline__ Rule rule_of(const SampleArgs& a, int64_t row) {
    float t = a.temperature, p = a.top_p, m = a.min_p;
    int32_t k = a.top_k;
    if (a.settings) {
        const float* s = a.settings + 4 * row;
        t = s[0]; p = s[2]; m = s[3];
        k = s[1] >= 1.0f ? (s[1] < (float)a.V ? (int32_t)s[1] : 0) : 0;
    }
    Rule r;
    r.greedy = t <= 0.0f;
    r.inv_t = 1.0 / (double)(t > 0.0f ? t : 1.0f);
    r.p = p < 1.0f ? (p > 0.0f ? (double)p : 0.0) : 1.0;                 // NaN: off
    r.log_m = m > 0.0f ? log((double)(m < 1.0f ? m : 1.0f)) : -HUGE_VAL;
    r.k = k >= 1 && k < a.V ? k : 0;
    return r;
}

constexpr double FIXED = 8796093022208.0;                                // 2^43
__device__ __forceinline__ float clean(float l) { return l != l ? -HUGE_VALF : l + 0.0f; }      // NaN -> -inf, -0 -> 0
// (l - max) / temperature, 0 for the maximum itself (also where that is infinite)
__device__ __forceinline__ double scaled(float l, float top, double inv_t) { return l == top ? 0.0 : ((double)l - (double)top) * inv_t; }
__device__ __forceinline__ u64 weight(double z) { return z > -31.0 ? (u64)(exp(z) * FIXED + 0.5) : 0; }
__device__ __forceinline__ float log_prob_of(double z, u64 total) { return (float)(z - log((double)total / FIXED)); }

__device__ __forceinline__ u64 shfl_u64(u64 v, int src, int width) {
    const int lo = __shfl((int)(uint32_t)v, src, width), hi = __shfl((int)(uint32_t)(v >> 32), src, width);
    return ((u64)(uint32_t)hi << 32) | (uint32_t)lo;
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int by, int width) {
    const int lo = __shfl_up((int)(uint32_t)v, by, width), hi = __shfl_up((int)(uint32_t)(v >> 32), by, width);
    return ((u64)(uint32_t)hi << 32) | (uint32_t)lo;
}

// -- up to 64 logits: L lanes per row ---------------------------------------------------------------------------------
template <typename T, int L>
__global__ __launch_bounds__(256) void sample_short_kernel(const SampleArgs a) {
    const int lane = threadIdx.x % L;
    const int64_t slot = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const bool live = slot < a.rows;
    const int64_t row = live ? slot : a.rows - 1;
    const Rule rule = rule_of(a, row);
    const float l = lane < a.V ? clean(to_f32(((const T*)a.logits)[row * a.ld + lane])) : -HUGE_VALF;
    float top = l;
#pragma unroll
    for (int o = L / 2; o > 0; o /= 2) top = fmaxf(top, __shfl_xor(top, o, L));
    const bool any = top > -HUGE_VALF;
    const double z = any ? scaled(l, top, rule.inv_t) : -HUGE_VAL;
    u64 w = rule.greedy ? 0 : weight(z);
    if (__any(rule.k > 0 || rule.p < 1.0)) {
        int rank = 0;
        u64 before = 0;
        for (int j = 0; j < L; ++j) {
            const float lj = __shfl(l, j, L);
            const u64 wj = shfl_u64(w, j, L);
            if (lj > l || (lj == l && j < lane)) { ++rank; before += wj; }
        }
        if (rule.k > 0 && rank >= rule.k) w = 0;
        u64 sum = w;
#pragma unroll
        for (int o = L / 2; o > 0; o /= 2) sum += shfl_u64(sum, (lane ^ o), L);
        if (rule.p < 1.0 && rank > 0 && !((double)before < rule.p * (double)sum)) w = 0;
    }
    if (z < rule.log_m) w = 0;
    u64 cum = w;
#pragma unroll
    for (int o = 1; o < L; o *= 2) { const u64 t = shfl_up_u64(cum, o, L); if (lane >= o) cum += t; }
    const u64 total = shfl_u64(cum, L - 1, L);
    float u = a.u[row];
    u = u > 0.0f ? (u < 1.0f ? u : 1.0f) : 0.0f;
    const double target = (double)u * (double)total;
    // the first lane past the target; if rounding or u = 1 leaves none, the last kept one
    const unsigned long long mask = L == 64 ? ~0ull : ((1ull << L) - 1) << (((threadIdx.x & 63) / L) * L);
    const unsigned long long hit = __ballot(rule.greedy ? l == top && any : w > 0 && (double)cum > target) & mask;
    const unsigned long long kept = __ballot(w > 0) & mask;
    int chosen = hit ? __ffsll((long long)hit) - 1 : kept ? 63 - __clzll((long long)kept) : -1;
    if (chosen >= 0) chosen %= L;
    if (live && lane == (chosen < 0 ? 0 : chosen)) {
        a.index[row] = any ? chosen : -1;
        a.log_prob[row] = !any ? -HUGE_VALF : rule.greedy ? 0.0f : log_prob_of(z, total);
    }
}

// -- longer rows: a workgroup per row ----------------------------------------------------------------------------------
constexpr int BINS = 2048, CAP = 2048;
constexpr double BINS_PER_NAT = 64.0;

__device__ __forceinline__ uint32_t key_of(float l) {                    // larger value, larger key
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ int bin_of(double z) {
    const double b = -z * BINS_PER_NAT;
    return b < (double)(BINS - 1) ? (int)b : BINS - 1;
}

template <int THREADS> struct Shared {
    uint32_t count[BINS];
    u64 mass[BINS];
    u64 list[CAP];                  // (~key << 32 | index): ascending = the order of the row
    u64 wave64[THREADS / 64];
    uint32_t wave32[THREADS / 64];
    u64 found_mass, found64;
    uint32_t n, found, found_count;
    float top;
};

// inclusive scan over the workgroup; *total = the sum
template <int THREADS> __device__ __forceinline__ u64 block_scan(u64 v, Shared<THREADS>& s, u64* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) { const u64 t = shfl_up_u64(v, o, 64); if (lane >= o) v += t; }
    __syncthreads();
    if (lane == 63) s.wave64[wave] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) { if (w < wave) before += s.wave64[w]; all += s.wave64[w]; }
    *total = all;
    return v + before;
}

// The kept prefix of the order ends with (key, index), both included.
struct Cut { uint32_t key, index; };
__device__ __forceinline__ bool inside(const Cut& c, uint32_t key, uint32_t i) { return key > c.key || (key == c.key && i <= c.index); }

template <typename T, int THREADS, class F>
__device__ __forceinline__ void each(const T* row, int32_t V, F&& f) {
    constexpr int CE = Chunk<T>::n;
    for (int32_t c = threadIdx.x * CE; c < V; c += THREADS * CE) {
        const Vec<T> v = load_part(row + c, (int64_t)V - c);
#pragma unroll
        for (int e = 0; e < CE; ++e) if (c + e < V) f(c + e, clean(to_f32(v.e[e])));
    }
}

// Where the running sum over the bins (counts, or masses) reaches `goal` first: the bin, and the count and mass before
// it.  by_count: first bin with count(0..b) >= goal_n; else the last bin with mass before it < goal_m (and not empty).
template <int THREADS>
__device__ __forceinline__ void find_bin(Shared<THREADS>& s, bool by_count, uint32_t goal_n, double goal_m, uint32_t& bin, uint32_t& n_before, u64& m_before) {
    constexpr int PER = BINS / THREADS;
    u64 n = 0, m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { n += s.count[threadIdx.x * PER + i]; m += s.mass[threadIdx.x * PER + i]; }
    u64 total;
    u64 cn = block_scan<THREADS>(n, s, &total) - n;
    u64 cm = block_scan<THREADS>(m, s, &total) - m;
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    u64 an = cn, am = cm;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = threadIdx.x * PER + i;
        const uint32_t c = s.count[b];
        const bool here = by_count ? an < goal_n && an + c >= goal_n : c > 0 && (double)am < goal_m;
        if (here) atomicMax(&s.found, (uint32_t)b);
        an += c; am += s.mass[b];
    }
    __syncthreads();
    bin = s.found;
    an = cn; am = cm;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t b = threadIdx.x * PER + i;
        if (b == bin) { s.found_count = (uint32_t)an; s.found_mass = am; }
        an += s.count[b]; am += s.mass[b];
    }
    __syncthreads();
    n_before = s.found_count; m_before = s.found_mass;
    __syncthreads();
}

// The last element of the shortest prefix of the order that holds goal_n elements (by_count), or that cannot lose its
// last element without its mass falling below goal_m, among the elements of linear bin `bin`; *mass = the mass up to
// and with it.  Elements of one bin are sorted in LDS; a bin with more than fits is cut by its keys first, down to a
// single value if need be, whose elements count by index.
template <typename T, int THREADS>
__device__ Cut resolve(Shared<THREADS>& s, const T* row, int32_t V, float top, double inv_t, uint32_t bin, bool by_count, uint32_t goal_n, double goal_m,
                       uint32_t n_before, u64 m_before, u64* mass) {
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    for (;;) {
        if (threadIdx.x == 0) { s.n = 0; s.found64 = ((u64)0) ; s.found = 0xFFFFFFFFu; s.found_count = 0; }
        __syncthreads();
        uint32_t kmin = 0xFFFFFFFFu, kmax = 0, mine = 0;
        each<T, THREADS>(row, V, [&](int32_t i, float l) {
            const uint32_t key = key_of(l);
            if (key < lo || key > hi || !(l > -HUGE_VALF) || bin_of(scaled(l, top, inv_t)) != (int)bin) return;
            kmin = key < kmin ? key : kmin; kmax = key > kmax ? key : kmax; ++mine;
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < CAP) s.list[at] = ((u64)(uint32_t)~key << 32) | (uint32_t)i;
        });
        if (mine) { atomicMin(&s.found, kmin); atomicMax(&s.found_count, kmax); }
        __syncthreads();
        const uint32_t n = s.n;
        kmin = s.found; kmax = s.found_count;
        __syncthreads();
        if (n <= CAP) {
            int size = 64;
            while (size < (int)n) size *= 2;
            for (int i = threadIdx.x; i < size; i += THREADS) if (i >= (int)n) s.list[i] = ~0ull;
            for (int k = 2; k <= size; k *= 2)
                for (int j = k / 2; j > 0; j /= 2) {
                    __syncthreads();
                    for (int i = threadIdx.x; i < size / 2; i += THREADS) {
                        const int x = 2 * j * (i / j) + i % j, y = x + j;
                        const u64 p = s.list[x], q = s.list[y];
                        if ((p > q) == ((x & k) == 0)) { s.list[x] = q; s.list[y] = p; }
                    }
                }
            __syncthreads();
            // mass before and up to every element, in order: each thread a run of them
            constexpr int PER = CAP / THREADS;
            u64 w[PER], sum = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = threadIdx.x * PER + i;
                uint32_t key = at < (int)n ? ~(uint32_t)(s.list[at] >> 32) : 0;
                const float l = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
                w[i] = at < (int)n ? weight(scaled(l, top, inv_t)) : 0;
                sum += w[i];
            }
            u64 total;
            u64 run = m_before + block_scan<THREADS>(sum, s, &total) - sum;
            if (threadIdx.x == 0) s.found = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t at = threadIdx.x * PER + i;
                const bool in = at < n && (by_count ? n_before + at < goal_n : n_before + at == 0 || (double)run < goal_m);
                if (in) atomicMax(&s.found, at);
                run += w[i];
            }
            __syncthreads();
            const uint32_t last = s.found;
            run = m_before + block_scan<THREADS>(sum, s, &total) - sum;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                run += w[i];
                if ((uint32_t)(threadIdx.x * PER + i) == last) s.found_mass = run;
            }
            __syncthreads();
            *mass = s.found_mass;
            const u64 e = s.list[last];
            __syncthreads();
            return Cut{~(uint32_t)(e >> 32), (uint32_t)e};
        }
        const float l_hi = __uint_as_float(kmax & 0x80000000u ? kmax & 0x7FFFFFFFu : ~kmax);
        if (kmin == kmax) {                         // one value: `take` of its elements, in index order
            const u64 w = weight(scaled(l_hi, top, inv_t));
            uint32_t take;
            if (by_count) take = goal_n - n_before;
            else {                                  // smallest t with m_before + t w >= goal_m
                const double want = goal_m - (double)m_before;
                take = w ? (uint32_t)ceil(want / (double)w) : n;
                while (take > 1 && !((double)(m_before + (u64)(take - 1) * w) < goal_m)) --take;
                while (take < n && (double)(m_before + (u64)take * w) < goal_m) ++take;
                if (take < 1) take = 1;
            }
            if (take > n) take = n;
            *mass = m_before + (u64)take * w;
            // the take-th element of this value: tiles of THREADS elements in index order
            uint32_t seen = 0;
            for (int32_t base = 0; base < V; base += THREADS) {
                const int32_t i = base + threadIdx.x;
                const bool is = i < V && key_of(clean(to_f32(row[i]))) == kmax;
                u64 tile;
                const u64 at = block_scan<THREADS>(is ? 1 : 0, s, &tile);
                if (is && seen + (uint32_t)at == take) s.found = (uint32_t)i;
                seen += (uint32_t)tile;
                __syncthreads();
                if (seen >= take) break;
            }
            const uint32_t last = s.found;
            __syncthreads();
            return Cut{kmax, last};
        }
        // histogram of [kmin, kmax] by key, largest first
        int shift = 0;
        while (((kmax - kmin) >> shift) >= BINS) ++shift;
        for (int b = threadIdx.x; b < BINS; b += THREADS) { s.count[b] = 0; s.mass[b] = 0; }
        __syncthreads();
        each<T, THREADS>(row, V, [&](int32_t, float l) {
            const uint32_t key = key_of(l);
            if (key < kmin || key > kmax || !(l > -HUGE_VALF)) return;
            const double z = scaled(l, top, inv_t);
            if (bin_of(z) != (int)bin) return;
            const int b = (int)((kmax - key) >> shift);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], weight(z));
        });
        __syncthreads();
        uint32_t b, nb;
        u64 mb;
        find_bin<THREADS>(s, by_count, by_count ? goal_n - n_before : 0, goal_m - (double)m_before, b, nb, mb);
        n_before += nb; m_before += mb;
        hi = kmax - (b << shift);
        const u64 span = ((u64)(b + 1) << shift) - 1;
        lo = kmax - kmin > span ? (uint32_t)(kmax - span) : kmin;
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(const SampleArgs a) {
    __shared__ Shared<THREADS> s;
    constexpr int CE = Chunk<T>::n;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* row = (const T*)a.logits + r * a.ld;
    const int32_t V = a.V;
    const Rule rule = rule_of(a, r);
    // maximum
    float top = -HUGE_VALF;
    each<T, THREADS>(row, V, [&](int32_t, float l) { top = fmaxf(top, l); });
#pragma unroll
    for (int o = 32; o > 0; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) s.wave32[wave] = __float_as_uint(top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, __uint_as_float(s.wave32[w]));
    __syncthreads();
    if (!(top > -HUGE_VALF)) {
        if (threadIdx.x == 0) { a.index[r] = -1; a.log_prob[r] = -HUGE_VALF; }
        return;
    }
    if (rule.greedy) {
        if (threadIdx.x == 0) s.found = 0xFFFFFFFFu;
        __syncthreads();
        uint32_t first = 0xFFFFFFFFu;
        each<T, THREADS>(row, V, [&](int32_t i, float l) { if (l == top && (uint32_t)i < first) first = (uint32_t)i; });
        if (first != 0xFFFFFFFFu) atomicMin(&s.found, first);
        __syncthreads();
        if (threadIdx.x == 0) { a.index[r] = s.found; a.log_prob[r] = 0.0f; }
        return;
    }
    Cut cut = {0, 0xFFFFFFFFu};
    if (rule.k > 0 || rule.p < 1.0) {
        for (int b = threadIdx.x; b < BINS; b += THREADS) { s.count[b] = 0; s.mass[b] = 0; }
        __syncthreads();
        u64 total = 0;
        each<T, THREADS>(row, V, [&](int32_t, float l) {
            if (!(l > -HUGE_VALF)) return;
            const double z = scaled(l, top, rule.inv_t);
            const int b = bin_of(z);
            atomicAdd(&s.count[b], 1u);
            if (rule.p < 1.0) { const u64 w = weight(z); if (w) atomicAdd(&s.mass[b], w); }
        });
        __syncthreads();
        u64 finite = 0, sum = 0;
        for (int b = threadIdx.x; b < BINS; b += THREADS) { finite += s.count[b]; sum += s.mass[b]; }
        block_scan<THREADS>(finite, s, &finite);
        block_scan<THREADS>(sum, s, &total);
        uint32_t b, nb;
        u64 mb;
        const bool limited = rule.k > 0 && (u64)rule.k < finite;
        if (limited) {
            find_bin<THREADS>(s, true, (uint32_t)rule.k, 0.0, b, nb, mb);
            // the bins may be needed again for top-p: resolve overwrites them only if the bin does not fit
            const bool fits = s.count[b] <= CAP;
            if (rule.p < 1.0 && !fits) {
                cut = resolve<T, THREADS>(s, row, V, top, rule.inv_t, b, true, (uint32_t)rule.k, 0.0, nb, mb, &total);
                for (int i = threadIdx.x; i < BINS; i += THREADS) { s.count[i] = 0; s.mass[i] = 0; }
                __syncthreads();
                each<T, THREADS>(row, V, [&](int32_t, float l) {
                    if (!(l > -HUGE_VALF)) return;
                    const double z = scaled(l, top, rule.inv_t);
                    atomicAdd(&s.count[bin_of(z)], 1u);
                    const u64 w = weight(z);
                    if (w) atomicAdd(&s.mass[bin_of(z)], w);
                });
                __syncthreads();
            } else {
                cut = resolve<T, THREADS>(s, row, V, top, rule.inv_t, b, true, (uint32_t)rule.k, 0.0, nb, mb, &total);
            }
        }
        if (rule.p < 1.0) {
            const double goal = rule.p * (double)total;
            find_bin<THREADS>(s, false, 0, goal > 1.0 ? goal : 1.0, b, nb, mb);
            u64 m;
            const Cut c = resolve<T, THREADS>(s, row, V, top, rule.inv_t, b, false, 0, goal, nb, mb, &m);
            if (c.key > cut.key || (c.key == cut.key && c.index < cut.index)) cut = c;
        }
    }
    // masses of the kept elements: wave w sums its run of the row, then the whole workgroup looks into the run of the draw
    auto kept = [&](int32_t i, float l, double z) { return l > -HUGE_VALF && !(z < rule.log_m) && inside(cut, key_of(l), (uint32_t)i); };
    constexpr int WAVES = THREADS / 64;
    const int32_t run = (V + WAVES * 64 * CE - 1) / (WAVES * 64 * CE) * (64 * CE);
    u64 sum = 0;
    for (int32_t c = wave * run + lane * CE; c < (wave + 1) * run && c < V; c += 64 * CE) {
        const Vec<T> v = load_part(row + c, (int64_t)V - c);
#pragma unroll
        for (int e = 0; e < CE; ++e) {
            if (c + e >= V) continue;
            const float l = clean(to_f32(v.e[e]));
            const double z = scaled(l, top, rule.inv_t);
            if (kept(c + e, l, z)) sum += weight(z);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o /= 2) sum += shfl_u64(sum, lane ^ o, 64);
    __syncthreads();
    if (lane == 0) s.wave64[wave] = sum;
    if (threadIdx.x == 0) { s.found = 0xFFFFFFFFu; s.found_count = 0; }
    __syncthreads();
    u64 total = 0, before = 0;
    int which = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += s.wave64[w];
    float u = a.u[r];
    u = u > 0.0f ? (u < 1.0f ? u : 1.0f) : 0.0f;
    double target = (double)u * (double)total;
    if (!(target < (double)total)) target = (double)(total - 1);          // u = 1, or rounded up: the last kept element
    {
        u64 cum = 0;
        bool hit = false;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const u64 m = s.wave64[w];
            if (!hit && (double)(cum + m) > target) { which = w; before = cum; hit = true; }
            cum += m;
        }
        if (!hit) {                                                        // masses beyond 2^53: the last wave with any
            cum = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { if (s.wave64[w]) { which = w; before = cum; } cum += s.wave64[w]; }
        }
    }
    const int32_t begin = which * run, end = begin + run < V ? begin + run : V;
    for (int32_t c0 = begin; c0 < end; c0 += THREADS * CE) {
        const int32_t c = c0 + threadIdx.x * CE;
        u64 w[CE], part = 0;
        const Vec<T> v = load_part(row + (c < end ? c : begin), c < end ? (int64_t)end - c : 0);
#pragma unroll
        for (int e = 0; e < CE; ++e) {
            w[e] = 0;
            if (c + e < end) {
                const float l = clean(to_f32(v.e[e]));
                const double z = scaled(l, top, rule.inv_t);
                if (kept(c + e, l, z)) w[e] = weight(z);
            }
            part += w[e];
        }
        u64 tile;
        u64 cum = before + block_scan<THREADS>(part, s, &tile) - part;
        uint32_t first = 0xFFFFFFFFu, last = 0;
#pragma unroll
        for (int e = CE - 1; e >= 0; --e) {
            u64 up = cum;
#pragma unroll
            for (int q = 0; q <= e; ++q) up += w[q];
            if (w[e] && (double)up > target) first = (uint32_t)(c + e);
            if (w[e] && last == 0) last = (uint32_t)(c + e) + 1;
        }
        if (first != 0xFFFFFFFFu) atomicMin(&s.found, first);
        if (last) atomicMax(&s.found_count, last);
        before += tile;
        __syncthreads();
        if (s.found != 0xFFFFFFFFu) break;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const int32_t i = s.found != 0xFFFFFFFFu ? (int32_t)s.found : (int32_t)s.found_count - 1;
        a.index[r] = i;
        a.log_prob[r] = log_prob_of(scaled(clean(to_f32(row[i])), top, rule.inv_t), total);
    }
}

template <typename T> int run(const SampleArgs& a, hipStream_t stream) {
#define MARL_SHORT(L) hipLaunchKernelGGL((sample_short_kernel<T, L>), dim3((unsigned)((a.rows + 256 / L - 1) / (256 / L))), dim3(256), 0, stream, a)
    if (a.V <= 4) MARL_SHORT(4);
    else if (a.V <= 8) MARL_SHORT(8);
    else if (a.V <= 16) MARL_SHORT(16);
    else if (a.V <= 32) MARL_SHORT(32);
    else if (a.V <= 64) MARL_SHORT(64);
#undef MARL_SHORT
    else if (a.V <= 4096) hipLaunchKernelGGL((sample_row_kernel<T, 256>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((sample_row_kernel<T, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

}  // namespace

extern "C" int marl_sample_logits(int32_t dtype, int64_t rows, int32_t V, const void* logits, int64_t ld, const float* u, float temperature,
                                  int32_t top_k, float top_p, float min_p, const float* settings, int64_t* index, float* log_prob, void* stream) {
    if (rows < 1 || V < 1 || !logits || !u || !index || !log_prob || dtype < MARL_F32 || dtype > MARL_F16 || (ld < V && rows > 1)) return MARL_EINVAL;
    if (!settings && (!(temperature >= 0.0f) || top_k < 0 || !(top_p > 0.0f) || !(min_p >= 0.0f && min_p <= 1.0f))) return MARL_EINVAL;
    if (V > MARL_MAX_CHOICES || rows > (1ll << 31) - 256) return MARL_EUNSUPPORTED;
    SampleArgs a = {logits, ld, rows, V, u, settings, temperature, top_p, min_p, top_k, index, log_prob};
    return MARL_BY_TYPE(dtype, run, a, (hipStream_t)stream);
}
