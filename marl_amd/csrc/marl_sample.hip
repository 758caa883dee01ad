// Draw of one index per row of logits, with temperature, top-k, top-p and min-p, from given uniform numbers:
//     z_i = l_i / temperature,  w_i = exp(z_i - max z);  order: larger logit first, equal ones by index
//     top-k   the first k of the order             top-p   of those, the shortest prefix whose mass reaches p of theirs
//     min-p   w_i >= min_p (of the largest)        draw    in index order, the first i with w_0 + .. + w_i > u * sum
// The kept set is always a prefix of the order, so it is described by its last element (value, index).  Weights are
// held as integers, w 2^42 rounded: their sums do not depend on the order of adding, so LDS atomics and any launch shape
// give the same index; sums are 64-bit integers (a row of 2^20 logits cannot overflow) or, up to 2048 logits, float64, which
// holds integers up to 2^53 exactly.  Weights below 2^-43 of the largest are 0: such an element is never drawn, for u = 0 or 1
// neither.  exp is evaluated in float64: an index depends on which side of a border a sum of many weights falls.
// NaN counts as -inf; +inf takes all the mass (several share it); a row without a finite or +inf logit gives index -1
// and log-probability -inf.  temperature <= 0: the first largest logit.
// Rows of up to 64 logits: a group of lanes per row, everything in registers.  Up to 2048: a wave per row, likewise; the
// borders of top-k and top-p are found by bisection over the bits of the ordered values, a count (ballots) or a sum each.
// Longer rows: a workgroup per row, which
// reads its row a few times (the first time from HBM, then from L2).  With a small top-k, twice: the maximum, and every
// thread's own two largest; k elements are above the k-th largest of those, so none below it can be among the first k;
// the few elements above are sorted in LDS and the rest happens there.  Otherwise: maximum; counts and masses over bins
// of a fraction of a nat below the maximum; the elements of the bin in which a border falls, sorted in LDS; the masses of
// the kept.
// Measured: 131072 x 4 float32 6.8 us; 256 x 131072 bf16 with settings per row 66 to 151 us, by whether some row's settings
// miss the short way for a small top-k (67 MB would take 13): one row's chain of passes on one CU is the bound, as for one
// row of 100003 (22 us).  65 to 2048 logits: 37 282 x 900 f16 with top-k 64 and top-p 188 us, top-p alone 234 (67 MB: 13): bisection.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

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

constexpr double FIXED = 4398046511104.0;                                // 2^42
__device__ __forceinline__ float clean(float l) { return l != l ? -HUGE_VALF : l + 0.0f; }      // NaN -> -inf, -0 -> 0
// (l - max) / temperature, 0 for the maximum itself (also where that is infinite)
__device__ __forceinline__ double scaled(float l, float top, double inv_t) { return l == top ? 0.0 : ((double)l - (double)top) * inv_t; }
// exp(z), z <= 0, in units of 2^-42, rounded to an integer (0 below -31 and for NaN): e^z = 2^(n / 64) e^r, |r| <= ln 2 / 128,
// with n / 64's fraction from a table of 64 and e^r from its series up to r^5 (rest below 4e-17).  The powers of two are
// added to the exponent; adding 1.5 2^52 rounds.  Half of the instructions of exp() and a conversion.
__constant__ const double kPow64[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951
};
constexpr double ROUND = 6755399441055744.0;                             // 1.5 2^52
__device__ __forceinline__ double weight_plus_round(double z, const double* pow64) {
    z = fmax(z, -40.0);                                                  // e^-40 rounds to 0; NaN becomes -40
    const double m = fma(z, 92.332482616893656759, ROUND);               // 64 / ln 2: the nearest integer in the low word
    const int n = (int)(uint32_t)__double_as_longlong(m);
    const double r = fma(m - ROUND, -0.010830424696249145, z);           // ln 2 / 64
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(r, e, 1.0 / 6.0);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    const long long v = __double_as_longlong(e * pow64[n & 63]) + ((long long)((n >> 6) + 42) << 52);
    return __longlong_as_double(v) + ROUND;
}
__device__ __forceinline__ double weight_f64(double z, const double* pow64) { return weight_plus_round(z, pow64) - ROUND; }
__device__ __forceinline__ u64 weight(double z, const double* pow64) {
    return (u64)(__double_as_longlong(weight_plus_round(z, pow64)) - __double_as_longlong(ROUND));
}
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
    u64 w = rule.greedy || !(z > -31.0) ? 0 : (u64)(exp(z) * FIXED + 0.5);
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

// -- up to 64 NE logits: a wave per row, lane i holds logits NE i .. NE i + NE - 1 -------------------------------------------
__device__ __forceinline__ uint32_t key_of(float l) {                    // larger value, larger key
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
// The kept prefix of the order ends with (key, index), both included.
struct Cut { uint32_t key, index; };
__device__ __forceinline__ bool inside(const Cut& c, uint32_t key, uint32_t i) { return key > c.key || (key == c.key && i <= c.index); }

__device__ __forceinline__ double target_of(const SampleArgs& a, int64_t r, double total) {
    float u = a.u[r];
    u = u > 0.0f ? (u < 1.0f ? u : 1.0f) : 0.0f;
    const double t = (double)u * total;
    return t < total ? t : total - 1.0;                  // u = 1, or rounded up: the last kept element
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o);
    return v;
}
// sum over the lanes below
__device__ __forceinline__ double wave_before(double v, int lane) {
    double s = v;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) { const double t = __shfl_up(s, o); if (lane >= o) s += t; }
    return s - v;
}

// bits of an ordered value below which all keys of one sign are equal: ones for negative values, zeros for others
template <typename T> struct LowBits { static constexpr int n = sizeof(T) == 4 ? 0 : std::is_same<T, bf16>::value ? 16 : 13; };

// the first `take` of the elements equal to `key`, in index order, are kept, those above all, the others lose their weight
template <int N> __device__ __forceinline__ void keep_above(const float (&l)[N], double (&w)[N], uint32_t key, int take, int lane) {
    int mine = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) mine += key_of(l[e]) == key;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) { const int t = __shfl_up(before, o); if (lane >= o) before += t; }
    before -= mine;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t k = key_of(l[e]);
        if (k < key || (k == key && before >= take)) w[e] = 0.0;
        before += k == key;
    }
}

// top-p, min-p and the draw among N weighted elements a lane, in index order over lanes and elements
template <typename T, int N, class Index>
__device__ __forceinline__ void finish_row(const SampleArgs& a, int64_t r, const Rule& rule, float top, const float (&l)[N], double (&w)[N], int lane, Index&& index_of) {
    constexpr int LOW = LowBits<T>::n;
    constexpr uint32_t ONES = (1u << LOW) - 1;
    if (rule.p < 1.0) {
        double sum = 0.0;
        uint32_t least = 0xFFFFFFFFu;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            sum += w[e];
            const uint32_t k = key_of(l[e]);
            if (w[e] > 0.0 && k < least) least = k;
        }
        double goal = rule.p * wave_sum(sum);
        goal = goal > 1.0 ? goal : 1.0;
#pragma unroll
        for (int o = 32; o > 0; o /= 2) { const uint32_t t = (uint32_t)__shfl_xor((int)least, o); least = t < least ? t : least; }
        // key: the largest with a mass of at least `goal` at or above it.  It lies between the smallest weighted value and
        // the maximum, whose common bits it shares.
        const uint32_t most = key_of(top), differ = most ^ least;
        const int high = differ ? 31 - __clz((int)differ) : -1;
        uint32_t key = high >= 31 ? 0 : most & ~((2u << (high < 0 ? 0 : high)) - 1u);
        if (high < 0) key = most;
#pragma unroll 1
        for (int bit = high; bit >= LOW; --bit) {
            const uint32_t c = key | (1u << bit);
            double m = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) m += (key_of(l[e]) | ONES) >= (c | ONES) ? w[e] : 0.0;
            if (wave_sum(m) >= goal) key = c;
        }
        double above = 0.0, one = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t k = key_of(l[e]) | ONES;
            above += k > (key | ONES) ? w[e] : 0.0;
            if (k == (key | ONES)) one = fmax(one, w[e]);
        }
        above = wave_sum(above);
#pragma unroll
        for (int o = 32; o > 0; o /= 2) one = fmax(one, __shfl_xor(one, o));
        // the smallest number of them that reaches the goal (at least one)
        double take = ceil((goal - above) / one);
        if (take > 1.0 && above + (take - 1.0) * one >= goal) take -= 1.0;
        if (above + take * one < goal) take += 1.0;
        keep_above<N>(l, w, key & 0x80000000u ? key & ~ONES : key | ONES, take > 1.0 ? (int)fmin(take, 4096.0) : 1, lane);
    }
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (scaled(l[e], top, rule.inv_t) < rule.log_m) w[e] = 0.0;
        sum += w[e];
    }
    double run = wave_before(sum, lane);
    const double total = __shfl(run + sum, 63), target = target_of(a, r, total);
    if (run <= target && run + sum > target) {
        bool found = false;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            run += w[e];
            if (!found && run > target) {
                found = true;
                a.index[r] = index_of(e);
                a.log_prob[r] = log_prob_of(scaled(l[e], top, rule.inv_t), (u64)total);
            }
        }
    }
}

template <typename T, int NE>
__global__ __launch_bounds__(256) void sample_wave_kernel(const SampleArgs a) {
    constexpr int CE = Chunk<T>::n;
    __shared__ double pow64[64];
    __shared__ float kept_l[4][64];
    __shared__ int kept_i[4][64];
    if (threadIdx.x < 64) pow64[threadIdx.x] = kPow64[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 4 + wave;
    if (r >= a.rows) return;
    const T* row = (const T*)a.logits + r * a.ld;
    const Rule rule = rule_of(a, r);
    const int at = lane * NE, left = a.V - at;
    float l[NE];
    if constexpr (NE >= CE) {
#pragma unroll
        for (int c = 0; c < NE; c += CE) {
            const Vec<T> v = load_clipped(row, (int64_t)at + c, (int64_t)a.V);
#pragma unroll
            for (int e = 0; e < CE; ++e) l[c + e] = left > c + e ? clean(to_f32(v.e[e])) : -HUGE_VALF;
        }
    } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) l[e] = left > e ? clean(to_f32(row[at + e])) : -HUGE_VALF;
    }
    float top = l[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) top = fmaxf(top, l[e]);
#pragma unroll
    for (int o = 32; o > 0; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    if (!(top > -HUGE_VALF)) {
        if (lane == 0) { a.index[r] = -1; a.log_prob[r] = -HUGE_VALF; }
        return;
    }
    if (rule.greedy) {
        int mine = NE;
#pragma unroll
        for (int e = NE - 1; e >= 0; --e) if (l[e] == top) mine = e;
        const unsigned long long any = __ballot(mine < NE);
        if (lane == __ffsll((long long)any) - 1) { a.index[r] = at + mine; a.log_prob[r] = 0.0f; }
        return;
    }
    double w[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) w[e] = 1.0;                // top-k needs no weights: a mark of what is left
    if (rule.k > 0) {
        constexpr int LOW = LowBits<T>::n;
        constexpr uint32_t ONES = (1u << LOW) - 1;
        uint32_t key = 0;                       // the largest with at least k elements at or above it, or one with exactly k
#pragma unroll 1
        for (int bit = 31; bit >= LOW; --bit) {
            const uint32_t c = key | (1u << bit);
            int n = 0;
#pragma unroll
            for (int e = 0; e < NE; ++e) n += __popcll(__ballot((key_of(l[e]) | ONES) >= (c | ONES)));
            if (n >= rule.k) key = c;
            if (n == rule.k) break;
        }
        int above = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) above += __popcll(__ballot((key_of(l[e]) | ONES) > (key | ONES)));
        keep_above<NE>(l, w, key & 0x80000000u ? key & ~ONES : key | ONES, rule.k - above, lane);
        if (rule.k <= 64) {                     // one element a lane from here on, still in index order
            int mine = 0;
#pragma unroll
            for (int e = 0; e < NE; ++e) mine += w[e] > 0.0;
            int to = mine;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) { const int t = __shfl_up(to, o); if (lane >= o) to += t; }
            const int n = __shfl(to, 63);
            to -= mine;
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (w[e] > 0.0) { kept_l[wave][to] = l[e]; kept_i[wave][to] = at + e; ++to; }
            __builtin_amdgcn_wave_barrier();            // one wave: its LDS accesses are done in order
            float l1[1] = {lane < n ? kept_l[wave][lane] : -HUGE_VALF};
            const int i1 = lane < n ? kept_i[wave][lane] : 0;
            double w1[1] = {weight_f64(scaled(l1[0], top, rule.inv_t), pow64)};
            finish_row<T, 1>(a, r, rule, top, l1, w1, lane, [&](int) { return i1; });
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) w[e] = w[e] > 0.0 ? weight_f64(scaled(l[e], top, rule.inv_t), pow64) : 0.0;
    finish_row<T, NE>(a, r, rule, top, l, w, lane, [&](int e) { return at + e; });
}

// -- longer rows: a workgroup per row ----------------------------------------------------------------------------------
// The workgroups: 1024 threads (one to a CU) for long rows if there are few, 256 for shorter rows and for many: what a row
// takes is mostly waiting, for its loads and at barriers (981 x 34 183 f16, top-k 64 and top-p: 74 us with 1024 threads).
// Where the two meet depends on the row's length: f16, 1024 : 256 threads, top-k 64 with top-p | top-p | no filter, us:
//     34 183 x  256     22 :  24  |    73 :  106  |   25 :  43          131 072 x  512     67 :  57  |   298 :  366  |  106 : 158
//     34 183 x  512     40 :  28  |   139 :  122  |   47 :  54          131 072 x 1024    124 :  89  |   590 :  549  |  202 : 254
//     34 183 x 1024     78 :  38  |   272 :  169  |   90 :  81          262 144 x 1024    214 : 200  |  1049 : 1072  |  377 : 502
// hence 256 from 512 rows on, up to 131 072 logits, and up to 8192 logits for any number of rows (9000 x 64: 18 : 17 | 42 : 45 |
// 16 : 18; x 384: 33 : 18 | 90 : 53 | 30 : 22).
// With 256, registers are held to six workgroups a CU; left free, the kernel takes more than 128 and two fit (same call,
// two : four : six a CU: 52 : 37 : 37 us; 4096 x 3000: 116 : 65 : 52; top-p alone, where six spill, 219 : 159 : 162).
template <int THREADS> struct Dim {
    static constexpr int BINS = THREADS == 1024 ? 2048 : 512;                    // bins
    static constexpr int CAP = THREADS == 1024 ? 2048 : 1024;                    // elements sorted at once
    static constexpr double PER_NAT = BINS / 32.0;                               // the bins cover 32 nats
};

template <int THREADS> __device__ __forceinline__ int bin_of(double z) {
    constexpr int BINS = Dim<THREADS>::BINS;
    const double b = -z * Dim<THREADS>::PER_NAT;
    return b < (double)(BINS - 1) ? (int)b : BINS - 1;
}

// Float32 bounds of the logits of a bin: none of bins up to `bin` lies below lower_edge, none of bins from `bin` on above
// upper_edge; what else lies between them is told apart by its bin.  The slack covers the roundings on the way: to float32, of
// the edge's size, and of the distance to the maximum, in float64, of the maximum's (which counts where the edge is next to 0).
__device__ __forceinline__ double edge_slack(double edge, float top) { return fabs(edge) * 0x1p-22 + fabs((double)top) * 0x1p-48 + 0x1p-126; }
template <int THREADS> __device__ __forceinline__ float lower_edge(int bin, float top, double inv_t) {
    if (bin >= Dim<THREADS>::BINS - 1) return -HUGE_VALF;
    const double edge = (double)top - (double)(bin + 1) / (Dim<THREADS>::PER_NAT * inv_t);
    return (float)(edge - edge_slack(edge, top));
}
template <int THREADS> __device__ __forceinline__ float upper_edge(int bin, float top, double inv_t) {
    if (bin <= 0) return HUGE_VALF;
    const double edge = (double)top - (double)bin / (Dim<THREADS>::PER_NAT * inv_t);
    return (float)(edge + edge_slack(edge, top));
}

template <int THREADS> struct Shared {
    double pow64[64];
    u64 mass[Dim<THREADS>::BINS];
    u64 list[Dim<THREADS>::CAP];    // (~key << 32 | index): ascending = the order of the row
    uint32_t count[Dim<THREADS>::BINS];
    u64 wave64[THREADS / 64];
    uint32_t wave32[THREADS / 64];
    u64 found_mass;
    uint32_t n, found, found_count;
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

// f(index, value) for every element of the row, four chunks per thread under way at a time
template <typename T, int THREADS, class F>
__device__ __forceinline__ void each(const T* row, int32_t V, F&& f) {
    constexpr int CE = Chunk<T>::n, TURN = THREADS * CE;
    int32_t c = threadIdx.x * CE;
    for (; c + 3 * TURN + CE <= V; c += 4 * TURN) {
        Vec<T> v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = load_chunk(row + c + q * TURN);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < CE; ++e) f(c + q * TURN + e, clean(to_f32(v[q].e[e])));
    }
    for (; c < V; c += TURN) {
        const Vec<T> v = load_part(row + c, (int64_t)V - c);
#pragma unroll
        for (int e = 0; e < CE; ++e) if (c + e < V) f(c + e, clean(to_f32(v.e[e])));
    }
}

// Where the running sum over the bins (counts, or masses) reaches `goal` first: the bin, and the count and mass before
// it.  by_count: first bin with count(0..b) >= goal_n; else the last bin of any mass with less than goal_m before it.
template <int THREADS>
__device__ __forceinline__ void find_bin(Shared<THREADS>& s, bool by_count, uint32_t goal_n, double goal_m, uint32_t& bin, uint32_t& n_before, u64& m_before) {
    constexpr int PER = Dim<THREADS>::BINS / THREADS;
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
        const bool here = by_count ? an < goal_n && an + c >= goal_n : s.mass[b] > 0 && (double)am < goal_m;
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

// ascending order of the first n elements of the list
template <int THREADS> __device__ __forceinline__ void sort_list(Shared<THREADS>& s, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = threadIdx.x; i < size; i += THREADS) if (i >= n) s.list[i] = ~0ull;
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
}

// The last element of the shortest prefix of the order that holds goal_n elements (by_count), or that cannot lose its
// last element without its mass falling below goal_m, among the elements of linear bin `bin`; *mass = the mass up to
// and with it.  Elements of one bin are sorted in LDS; a bin with more than fits is cut by its keys first, down to a
// single value if need be, whose elements count by index.
template <typename T, int THREADS>
__device__ __noinline__ Cut resolve(Shared<THREADS>& s, const T* row, int32_t V, float top, double inv_t, uint32_t bin, bool by_count, uint32_t goal_n, double goal_m,
                                    uint32_t n_before, u64 m_before, u64* mass) {
    constexpr int BINS = Dim<THREADS>::BINS, CAP = Dim<THREADS>::CAP;
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    // cheap bounds first: most of the row is outside of the bin (+inf logits, whose distances are not numbers: no bounds)
    const bool bounded = fabsf(top) < HUGE_VALF;
    const float floor_ = bounded ? lower_edge<THREADS>((int)bin, top, inv_t) : -HUGE_VALF;
    const float ceiling = bounded ? upper_edge<THREADS>((int)bin, top, inv_t) : HUGE_VALF;
    for (;;) {
        if (threadIdx.x == 0) { s.n = 0; s.found = 0xFFFFFFFFu; s.found_count = 0; }
        __syncthreads();
        uint32_t kmin = 0xFFFFFFFFu, kmax = 0, mine = 0;
        each<T, THREADS>(row, V, [&](int32_t i, float l) {
            if (!(l >= floor_ && l <= ceiling)) return;
            const uint32_t key = key_of(l);
            if (key < lo || key > hi || !(l > -HUGE_VALF) || bin_of<THREADS>(scaled(l, top, inv_t)) != (int)bin) return;
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
            sort_list<THREADS>(s, (int)n);
            // mass before and up to every element, in order: each thread a run of them
            constexpr int PER = CAP / THREADS;
            u64 w[PER], sum = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = threadIdx.x * PER + i;
                w[i] = at < (int)n ? weight(scaled(value_of(~(uint32_t)(s.list[at] >> 32)), top, inv_t), s.pow64) : 0;
                sum += w[i];
            }
            u64 total;
            u64 run = m_before + block_scan<THREADS>(sum, s, &total) - sum;
            if (threadIdx.x == 0) s.found = 0;
            __syncthreads();
            u64 upto[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t at = threadIdx.x * PER + i;
                const bool in = at < n && (by_count ? n_before + at < goal_n : at == 0 || (double)run < goal_m);
                if (in) atomicMax(&s.found, at);
                upto[i] = run += w[i];
            }
            __syncthreads();
            const uint32_t last = s.found;
#pragma unroll
            for (int i = 0; i < PER; ++i) if ((uint32_t)(threadIdx.x * PER + i) == last) s.found_mass = upto[i];
            __syncthreads();
            *mass = s.found_mass;
            const u64 e = s.list[last];
            __syncthreads();
            return Cut{~(uint32_t)(e >> 32), (uint32_t)e};
        }
        if (kmin == kmax) {                         // one value: `take` of its elements, in index order
            const u64 w = weight(scaled(value_of(kmax), top, inv_t), s.pow64);
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
            if (!(l >= floor_ && l <= ceiling)) return;
            const uint32_t key = key_of(l);
            if (key < kmin || key > kmax || !(l > -HUGE_VALF)) return;
            const double z = scaled(l, top, inv_t);
            if (bin_of<THREADS>(z) != (int)bin) return;
            const int b = (int)((kmax - key) >> shift);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], weight(z, s.pow64));
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

// counts, masses or both of the row over the linear bins
template <typename T, int THREADS>
__device__ __noinline__ void histogram(Shared<THREADS>& s, const T* row, int32_t V, float top, double inv_t, bool counts, bool masses) {
    for (int b = threadIdx.x; b < Dim<THREADS>::BINS; b += THREADS) { s.count[b] = 0; s.mass[b] = 0; }
    __syncthreads();
    each<T, THREADS>(row, V, [&](int32_t, float l) {
        if (!(l > -HUGE_VALF)) return;
        const double z = scaled(l, top, inv_t);
        const int b = bin_of<THREADS>(z);
        if (counts) atomicAdd(&s.count[b], 1u);
        if (masses) { const u64 w = weight(z, s.pow64); if (w) atomicAdd(&s.mass[b], w); }
    });
    __syncthreads();
}

// where the kept prefix ends under top-k and top-p
template <typename T, int THREADS>
__device__ __noinline__ Cut cut_of(Shared<THREADS>& s, const T* row, int32_t V, float top, const Rule& rule) {
    Cut cut = {0, 0xFFFFFFFFu};
    histogram<T, THREADS>(s, row, V, top, rule.inv_t, rule.k > 0, rule.p < 1.0);
    u64 finite = 0, total = 0;
    for (int b = threadIdx.x; b < Dim<THREADS>::BINS; b += THREADS) { finite += s.count[b]; total += s.mass[b]; }
    block_scan<THREADS>(finite, s, &finite);
    block_scan<THREADS>(total, s, &total);
    uint32_t b, nb;
    u64 mb;
    if (rule.k > 0 && (u64)rule.k < finite) {
        find_bin<THREADS>(s, true, (uint32_t)rule.k, 0.0, b, nb, mb);
        const bool fits = s.count[b] <= Dim<THREADS>::CAP;              // else resolve() overwrites the bins
        cut = resolve<T, THREADS>(s, row, V, top, rule.inv_t, b, true, (uint32_t)rule.k, 0.0, nb, mb, &total);
        if (rule.p < 1.0 && !fits) histogram<T, THREADS>(s, row, V, top, rule.inv_t, false, true);
    }
    if (rule.p < 1.0) {
        const double goal = rule.p * (double)total;
        find_bin<THREADS>(s, false, 0, goal > 1.0 ? goal : 1.0, b, nb, mb);
        u64 m;
        // (counts may be absent or stale here: resolve() needs none, its bin has less than `goal` before it)
        const Cut c = resolve<T, THREADS>(s, row, V, top, rule.inv_t, b, false, 0, goal, 0, mb, &m);
        if (c.key > cut.key || (c.key == cut.key && c.index < cut.index)) cut = c;
    }
    return cut;
}

// Rows with top-k up to CAP / 4: true if the draw was made.  `mine`, `mine2`: the thread's own two largest.
template <typename T, int THREADS>
__device__ __forceinline__ bool draw_from_first_k(Shared<THREADS>& s, const SampleArgs& a, int64_t r, const T* row, float top, float mine, float mine2, const Rule& rule) {
    constexpr int BINS = Dim<THREADS>::BINS, CAP = Dim<THREADS>::CAP, PER = CAP / THREADS;
    const int32_t V = a.V;
    for (int b = threadIdx.x; b < BINS; b += THREADS) { s.count[b] = 0; s.mass[b] = 0; }
    if (threadIdx.x == 0) { s.n = 0; s.found = BINS; }
    __syncthreads();
    if (mine > -HUGE_VALF) atomicAdd(&s.count[bin_of<THREADS>(scaled(mine, top, rule.inv_t))], 1u);
    if (mine2 > -HUGE_VALF) atomicAdd(&s.count[bin_of<THREADS>(scaled(mine2, top, rule.inv_t))], 1u);
    __syncthreads();
    {   // the bin of the k-th largest of those
        u64 n = 0, all;
#pragma unroll
        for (int i = 0; i < BINS / THREADS; ++i) n += s.count[threadIdx.x * (BINS / THREADS) + i];
        u64 before = block_scan<THREADS>(n, s, &all) - n;
#pragma unroll
        for (int i = 0; i < BINS / THREADS; ++i) {
            const uint32_t b = threadIdx.x * (BINS / THREADS) + i, c = s.count[b];
            if (before < (u64)rule.k && before + c >= (u64)rule.k) s.found = b;
            before += c;
        }
    }
    __syncthreads();
    const uint32_t bin = s.found;
    if (bin >= BINS - 1) return false;              // fewer than k of them, or in the last bin, which has no lower edge
    // no element of bins 0 .. bin lies below this
    const float limit = lower_edge<THREADS>(bin, top, rule.inv_t);
    each<T, THREADS>(row, V, [&](int32_t i, float l) {
        if (l >= limit) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < CAP) s.list[at] = ((u64)(uint32_t)~key_of(l) << 32) | (uint32_t)i;
        }
    });
    __syncthreads();
    const int n = (int)s.n;
    if (n > CAP) return false;
    sort_list<THREADS>(s, n);
    const int first = n < rule.k ? n : rule.k;
    uint32_t index[PER];
    double z[PER];
    u64 w[PER], sum = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = threadIdx.x * PER + i;
        const u64 e = at < first ? s.list[at] : 0;
        index[i] = (uint32_t)e;
        z[i] = at < first ? scaled(value_of(~(uint32_t)(e >> 32)), top, rule.inv_t) : -HUGE_VAL;
        w[i] = weight(z[i], s.pow64);
        sum += w[i];
    }
    u64 before = block_scan<THREADS>(sum, s, &all) - sum;
    const double goal = rule.p * (double)all;
    sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const u64 own = w[i];
        if ((rule.p < 1.0 && threadIdx.x * PER + i > 0 && !((double)before < goal)) || z[i] < rule.log_m) w[i] = 0;
        before += own;
        sum += w[i];
    }
    // index order: masses by ranges of indices (s.mass is clear), then inside the range of the draw
    const uint32_t width = (uint32_t)(V + BINS - 1) / BINS;
#pragma unroll
    for (int i = 0; i < PER; ++i) if (w[i]) atomicAdd(&s.mass[index[i] / width], w[i]);
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    u64 m = 0, total;
#pragma unroll
    for (int i = 0; i < BINS / THREADS; ++i) m += s.mass[threadIdx.x * (BINS / THREADS) + i];
    u64 run = block_scan<THREADS>(m, s, &total) - m;
    const double target = target_of(a, r, (double)total);
#pragma unroll
    for (int i = 0; i < BINS / THREADS; ++i) {
        const uint32_t b = threadIdx.x * (BINS / THREADS) + i;
        const u64 c = s.mass[b];
        if ((double)run <= target && (double)(run + c) > target) { s.found = b; s.found_mass = run; }
        run += c;
    }
    __syncthreads();
    const uint32_t range = s.found;
    const u64 at_range = s.found_mass;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (w[i] && index[i] / width == range) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            s.list[at] = index[i];
            s.mass[at] = w[i];
        }
    __syncthreads();
    const int in_range = (int)s.n;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (w[i] && index[i] / width == range) {
            u64 low = at_range;
            for (int j = 0; j < in_range; ++j) if (s.list[j] < index[i]) low += s.mass[j];
            if ((double)low <= target && (double)(low + w[i]) > target) {
                a.index[r] = index[i];
                a.log_prob[r] = log_prob_of(z[i], total);
            }
        }
    return true;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? 6 : 4) void sample_row_kernel(const SampleArgs a) {
    __shared__ Shared<THREADS> s;
    constexpr int CE = Chunk<T>::n;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* row = (const T*)a.logits + r * a.ld;
    const int32_t V = a.V;
    const Rule rule = rule_of(a, r);
    if (threadIdx.x < 64) s.pow64[threadIdx.x] = kPow64[threadIdx.x];
    // maximum
    float mine = -HUGE_VALF, mine2 = -HUGE_VALF;
    each<T, THREADS>(row, V, [&](int32_t, float l) { mine2 = fmaxf(mine2, fminf(mine, l)); mine = fmaxf(mine, l); });
    float top = mine;
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
    if (rule.k > 0 && rule.k <= Dim<THREADS>::CAP / 4 && fabsf(top) < HUGE_VALF) {
        if (draw_from_first_k<T, THREADS>(s, a, r, row, top, mine, mine2, rule)) return;
        __syncthreads();
    }
    const Cut cut = rule.k > 0 || rule.p < 1.0 ? cut_of<T, THREADS>(s, row, V, top, rule) : Cut{0, 0xFFFFFFFFu};
    // masses of the kept elements: wave w sums its run of the row, then the whole workgroup looks into the run of the draw
    auto kept_weight = [&](int32_t i, float l) -> u64 {
        if (!(l > -HUGE_VALF) || !inside(cut, key_of(l), (uint32_t)i)) return 0;
        const double z = scaled(l, top, rule.inv_t);
        return z < rule.log_m ? 0 : weight(z, s.pow64);
    };
    constexpr int WAVES = THREADS / 64;
    const int32_t run = (V + WAVES * 64 * CE - 1) / (WAVES * 64 * CE) * (64 * CE);
    u64 sum = 0;
    if (cut.key == 0 && !(rule.log_m > -HUGE_VAL) && fabsf(top) < HUGE_VALF) {       // nothing is filtered
        double part = 0.0;                        // exact: at most 2^10 weights of at most 2^42
        const int32_t stop = (wave + 1) * run < V ? (wave + 1) * run : V;
        int32_t c = wave * run + lane * CE;
        for (; c + 192 * CE + CE <= stop; c += 256 * CE) {
            Vec<T> v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = load_chunk(row + c + 64 * CE * q);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < CE; ++e) part += weight_f64(((double)clean(to_f32(v[q].e[e])) - (double)top) * rule.inv_t, s.pow64);
        }
        for (; c < stop; c += 64 * CE) {
            const Vec<T> v = load_part(row + c, (int64_t)V - c);
#pragma unroll
            for (int e = 0; e < CE; ++e) if (c + e < V) part += weight_f64(((double)clean(to_f32(v.e[e])) - (double)top) * rule.inv_t, s.pow64);
        }
        sum = (u64)part;
    } else {
        for (int32_t c = wave * run + lane * CE; c < (wave + 1) * run && c < V; c += 64 * CE) {
            const Vec<T> v = load_part(row + c, (int64_t)V - c);
#pragma unroll
            for (int e = 0; e < CE; ++e)
                if (c + e < V) sum += kept_weight(c + e, clean(to_f32(v.e[e])));
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
    const double target = target_of(a, r, (double)total);
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
            w[e] = c + e < end ? kept_weight(c + e, clean(to_f32(v.e[e]))) : 0;
            part += w[e];
        }
        u64 tile;
        u64 cum = before + block_scan<THREADS>(part, s, &tile) - part;
        uint32_t first = 0xFFFFFFFFu, last = 0;
#pragma unroll
        for (int e = 0; e < CE; ++e) {
            cum += w[e];
            if (w[e] && first == 0xFFFFFFFFu && (double)cum > target) first = (uint32_t)(c + e);
            if (w[e]) last = (uint32_t)(c + e) + 1;
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

template <typename T> void launch(const SampleArgs& a, hipStream_t stream) {
#define MARL_SHORT(L) hipLaunchKernelGGL((sample_short_kernel<T, L>), dim3((unsigned)((a.rows + 256 / L - 1) / (256 / L))), dim3(256), 0, stream, a)
#define MARL_WAVE(NE) hipLaunchKernelGGL((sample_wave_kernel<T, NE>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, stream, a)
    if (a.V <= 4) MARL_SHORT(4);
    else if (a.V <= 8) MARL_SHORT(8);
    else if (a.V <= 16) MARL_SHORT(16);
    else if (a.V <= 32) MARL_SHORT(32);
    else if (a.V <= 64) MARL_SHORT(64);
    else if (a.V <= 128) MARL_WAVE(2);
    else if (a.V <= 256) MARL_WAVE(4);
    else if (a.V <= 512) MARL_WAVE(8);
    else if (a.V <= 1024) MARL_WAVE(16);
    else if (a.V <= 2048) MARL_WAVE(32);
    else if (a.V <= 8192 || (a.rows >= 512 && a.V <= 131072)) hipLaunchKernelGGL((sample_row_kernel<T, 256>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((sample_row_kernel<T, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, stream, a);
#undef MARL_SHORT
#undef MARL_WAVE
}

template <typename T> int run(const SampleArgs& all, hipStream_t stream) {
    constexpr int64_t MOST = 1 << 21;              // rows of a launch: its threads stay below 2^32
    for (int64_t first = 0; first < all.rows; first += MOST) {
        SampleArgs a = all;
        a.logits = (const T*)all.logits + first * all.ld;
        a.rows = all.rows - first < MOST ? all.rows - first : MOST;
        a.u += first; a.index += first; a.log_prob += first;
        if (a.settings) a.settings += 4 * first;
        launch<T>(a, stream);
    }
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
