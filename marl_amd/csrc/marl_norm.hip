// The norms around a residual block with its gate and residual scale, one pass over each row:
//     o = N(block; w_post)      y = scale x + gate o      n = N(y; w_pre)
// N(v; w) = w (v - m) r with m = mean (kind "layer") or 0 ("rms") and r = 1 / sqrt(mean((v - m)^2) + eps); gate is absent,
// one value per channel or one per element.  Backward, with hats for the normalised values, t = gy + N'(gn w_pre; y):
//     dx = scale t,  dgate = t o,  dblock = N'(t gate w_post; block),  dw_post = sum t gate block^,  dw_pre = sum gn y^,
//     N'(g; v) = r (g - mean(g) [layer only] - v^ mean(g v^)).
// Bandwidth bound: a row lives in the registers of its threads (16 lanes to 1024 threads, one 16-byte chunk each up to 512
// chunks, two or four beyond), so that forward reads x and block once and backward gy, gn, x and block once.  Workgroups stay
// and take row after row: the next row's chunks are under way while the sums of this one cross the waves, and the weights' chunks
// are held throughout.  Sums and statistics are float32; y is
// normalised before it is rounded.  m and r of both norms are kept (16 bytes a row), and backward computes y from x and block
// again: taken from memory, y has been rounded, and with the statistics of the unrounded row that leaves an error of half a
// step of y, times r, in y^ (a row of mean 64 and spread 1 in bf16: 0.14), at the same bytes.  The column sums of backward
// stay in registers over a workgroup's rows, go to a partial row per workgroup and are added by a second launch in a fixed
// order (no atomics: results do not vary from run to run).
// Measured: forward 131072 x 128 float32 43 us (6.2 TB/s), 16384 x 4096 bf16 102 us (5.3); backward 80 us (5.0) and, with a
// channel gate, 211 us (3.8) and 6 us for the columns' sum: 154 registers, three waves a SIMD.  Rows of more than 1024 chunks
// do not fit: backward spills 35 to 326 registers a thread and is bound by that traffic (4096 x 8192 float32 473 us, 1.7 TB/s;
// 2048 x 16384 float32 1007, 0.8; 4096 x 16384 bf16 1192, 0.7), forward only from 8193 float32 on (2048 x 16384: 163 us, 3.3).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "marl_env.h"
#include "marl_net.h"
#include "marl_types.h"

extern "C" __attribute__((visibility("hidden"))) void marl_note_hip_error(int err);     // marl_env.hip

namespace {

using namespace marl_types;

enum Gate { NO_GATE, CHANNEL_GATE, ROW_GATE };

struct NormArgs {
    const void *x, *block, *w_post, *w_pre, *gate;
    int64_t ldx, ldb, ldg;
    void *y, *n;
    float* stats;                     // [rows][4]: mean and rstd of block, of y
    const void *gy, *gn;              // backward
    int64_t ldgy, ldgn;
    void *dx, *dblock, *dgate_rows;   // contiguous [rows][d]
    float* partial;                   // [blocks][3][d]: dw_post, dw_pre, dgate per channel
    int64_t rows;
    int32_t d;
    int32_t layer, gate_kind;
    float scale, eps;
};

// Threads of one row: LANES of a wave (16, 32 or 64) or LANES / 64 waves.
template <int LANES> struct Row {
    static constexpr int THREADS = LANES < 256 ? 256 : LANES;
    static constexpr int ROWS = THREADS / LANES;                 // rows a workgroup works on at a time
    // sums of two values over the row's threads
    static __device__ __forceinline__ void sum2(float& a, float& b, float* scratch) {
        constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
        for (int o = W / 2; o > 0; o /= 2) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
        if constexpr (LANES > 64) {
            constexpr int WAVES = LANES / 64;
            float* mine = scratch + threadIdx.x / LANES * (2 * WAVES);
            __syncthreads();                                      // the last sum's values have been read
            if ((threadIdx.x & 63) == 0) *(float2*)(mine + 2 * ((threadIdx.x % LANES) / 64)) = make_float2(a, b);
            __syncthreads();
            a = b = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { a += mine[2 * w]; b += mine[2 * w + 1]; }
        }
    }
};

template <typename T, int NV> struct Regs { float v[NV][Chunk<T>::n]; };
template <typename T, int NV> struct Packed { Vec<T> v[NV]; };           // as in memory

// Rows of whole chunks; rows whose last chunk is ragged; rows shorter than a chunk.  Loads never branch on the data's
// end (a load whose result is merged with another path's is waited for on the spot): a chunk past the end repeats the
// last whole one, and the ragged chunk is the last CE elements of the row, moved to its place when it is used.
enum Width { WHOLE, RAGGED, TINY };

template <typename T, int NV, int LANES, int WIDTH>
__device__ __forceinline__ void load_row(Packed<T, NV>& out, const T* row, int32_t d, int lane) {
    constexpr int CE = Chunk<T>::n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * LANES + lane) * CE;
        if constexpr (WIDTH == TINY) out.v[i] = load_part(row, c == 0 ? d : 0);
        else out.v[i] = load_chunk(row + (c < d - CE ? c : d - CE));
    }
}
// the values of chunk i in float32, zero from d on
template <typename T, int NV, int LANES, int WIDTH>
__device__ __forceinline__ void unpack(float (&out)[Chunk<T>::n], const Packed<T, NV>& in, int i, int32_t d, int lane, bool live = true) {
    constexpr int CE = Chunk<T>::n;
    const int c = (i * LANES + lane) * CE;
    Vec<T> v = in.v[i];
    if constexpr (WIDTH == RAGGED) {              // the first element wanted is number c - (d - CE) of those loaded
        const int by = c > d - CE ? c - (d - CE) : 0;
#pragma unroll
        for (int step = 1; step < CE; step *= 2)
#pragma unroll
            for (int e = 0; e < CE; ++e) v.e[e] = (by & step) && e + step < CE ? v.e[e + step] : v.e[e];
    }
#pragma unroll
    for (int e = 0; e < CE; ++e) out[e] = live && c + e < d ? to_f32(v.e[e]) : 0.0f;
}
template <typename T, int NV, int LANES>
__device__ __forceinline__ void store_row(T* row, const Regs<T, NV>& in, int32_t d, int lane, bool live) {
    constexpr int CE = Chunk<T>::n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * LANES + lane) * CE;
        if (!live || c >= d) continue;
        Vec<T> t;
#pragma unroll
        for (int e = 0; e < CE; ++e) t.e[e] = from_f32<T>(in.v[i][e]);
        store_part(row + c, t, (int64_t)d - c);
    }
}

#define FOR_ROW(i, e)                       \
    _Pragma("unroll") for (int i = 0; i < NV; ++i) \
    _Pragma("unroll") for (int e = 0; e < Chunk<T>::n; ++e)

// mean (0 for rms) and 1 / sqrt(variance + eps) of a row
template <typename T, int NV, int LANES>
__device__ __forceinline__ void row_stats(const Regs<T, NV>& v, int32_t d, int lane, bool layer, float eps, float* scratch, float& m, float& r) {
    float s = 0.0f, zero = 0.0f;
    m = 0.0f;
    if (layer) {
        FOR_ROW(i, e) s += v.v[i][e];
        Row<LANES>::sum2(s, zero, scratch);
        m = s / (float)d;
    }
    float q = 0.0f;
    FOR_ROW(i, e) {
        const float t = (i * LANES + lane) * Chunk<T>::n + e < d ? v.v[i][e] - m : 0.0f;
        q = fmaf(t, t, q);
    }
    zero = 0.0f;
    Row<LANES>::sum2(q, zero, scratch);
    r = 1.0f / sqrtf(q / (float)d + eps);
}

template <typename T, int NV, int LANES, int WIDTH>
__global__ __launch_bounds__(Row<LANES>::THREADS) void residual_norm_kernel(const NormArgs a) {
    using R = Row<LANES>;
    using P = Packed<T, NV>;
    __shared__ float scratch[32];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const int32_t d = a.d;
    P wpost, wpre, gate, nb, nx;
    load_row<T, NV, LANES, WIDTH>(wpost, (const T*)a.w_post, d, lane);
    load_row<T, NV, LANES, WIDTH>(wpre, (const T*)a.w_pre, d, lane);
    if (a.gate_kind == CHANNEL_GATE) load_row<T, NV, LANES, WIDTH>(gate, (const T*)a.gate, d, lane);
    auto fetch = [&](int64_t r0, P& b, P& x) {
        const int64_t r = r0 + slot < a.rows ? r0 + slot : a.rows - 1;
        load_row<T, NV, LANES, WIDTH>(b, (const T*)a.block + r * a.ldb, d, lane);
        load_row<T, NV, LANES, WIDTH>(x, (const T*)a.x + r * a.ldx, d, lane);
    };
    const int64_t turn = (int64_t)gridDim.x * R::ROWS;
    int64_t r0 = (int64_t)blockIdx.x * R::ROWS;
    fetch(r0, nb, nx);
    for (; r0 < a.rows; r0 += turn) {
        const bool live = r0 + slot < a.rows;
        const int64_t r = live ? r0 + slot : a.rows - 1;
        const P x = nx;
        Regs<T, NV> b, y;
        float w[Chunk<T>::n];
#pragma unroll
        for (int i = 0; i < NV; ++i) unpack<T, NV, LANES, WIDTH>(b.v[i], nb, i, d, lane);
        if (r0 + turn < a.rows) fetch(r0 + turn, nb, nx);
        float mb, rb, my, ry;
        row_stats<T, NV, LANES>(b, d, lane, a.layer, a.eps, scratch, mb, rb);
        if (a.gate_kind == ROW_GATE) load_row<T, NV, LANES, WIDTH>(gate, (const T*)a.gate + r * a.ldg, d, lane);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            constexpr int CE = Chunk<T>::n;
            unpack<T, NV, LANES, WIDTH>(w, wpost, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) b.v[i][e] = (b.v[i][e] - mb) * rb * w[e];
            if (a.gate_kind != NO_GATE) {
                unpack<T, NV, LANES, WIDTH>(w, gate, i, d, lane);
#pragma unroll
                for (int e = 0; e < CE; ++e) b.v[i][e] *= w[e];
            }
            unpack<T, NV, LANES, WIDTH>(y.v[i], x, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) y.v[i][e] = fmaf(a.scale, y.v[i][e], b.v[i][e]);
        }
        store_row<T, NV, LANES>((T*)a.y + r * d, y, d, lane, live);
        row_stats<T, NV, LANES>(y, d, lane, a.layer, a.eps, scratch, my, ry);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T, NV, LANES, WIDTH>(w, wpre, i, d, lane);
#pragma unroll
            for (int e = 0; e < Chunk<T>::n; ++e) y.v[i][e] = (y.v[i][e] - my) * ry * w[e];
        }
        store_row<T, NV, LANES>((T*)a.n + r * d, y, d, lane, live);
        if (a.stats && live && lane == 0) *(float4*)(a.stats + 4 * r) = make_float4(mb, rb, my, ry);
    }
}

// g := r (g - mean(g) - hat mean(g hat)), hat in `h`; the elements beyond d are zero in both
template <typename T, int NV, int LANES>
__device__ __forceinline__ void norm_back(Regs<T, NV>& g, const Regs<T, NV>& h, int32_t d, bool layer, float r, float* scratch) {
    float s = 0.0f, p = 0.0f;
    FOR_ROW(i, e) { s += g.v[i][e]; p = fmaf(g.v[i][e], h.v[i][e], p); }
    Row<LANES>::sum2(s, p, scratch);
    s = layer ? s / (float)d : 0.0f;
    p /= (float)d;
    FOR_ROW(i, e) g.v[i][e] = r * (g.v[i][e] - s - h.v[i][e] * p);
}

// GATE is known at compile time: without a channel gate its column sums take no registers, without any gate neither its chunks.
template <typename T, int NV, int LANES, int WIDTH, int GATE>
__global__ __launch_bounds__(Row<LANES>::THREADS) void residual_norm_backward_kernel(const NormArgs a) {
    using R = Row<LANES>;
    constexpr int CE = Chunk<T>::n;
    __shared__ float scratch[32];
    __shared__ float columns[R::ROWS > 1 ? R::THREADS * NV * CE : 1];       // one sum at a time
    using P = Packed<T, NV>;
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const int32_t d = a.d;
    Regs<T, NV> spost = {}, spre = {}, sgate = {};
    P wpost, wpre, gate, nx, ngn, ngy, nb, ngate;
    float4 nst;
    load_row<T, NV, LANES, WIDTH>(wpost, (const T*)a.w_post, d, lane);
    load_row<T, NV, LANES, WIDTH>(wpre, (const T*)a.w_pre, d, lane);
    if constexpr (GATE == CHANNEL_GATE) load_row<T, NV, LANES, WIDTH>(gate, (const T*)a.gate, d, lane);
    auto fetch = [&](int64_t r0) {
        const int64_t r = r0 + slot < a.rows ? r0 + slot : a.rows - 1;
        nst = *(const float4*)(a.stats + 4 * r);
        load_row<T, NV, LANES, WIDTH>(nx, (const T*)a.x + r * a.ldx, d, lane);
        load_row<T, NV, LANES, WIDTH>(nb, (const T*)a.block + r * a.ldb, d, lane);
        if (a.gn) load_row<T, NV, LANES, WIDTH>(ngn, (const T*)a.gn + r * a.ldgn, d, lane);
        if (a.gy) load_row<T, NV, LANES, WIDTH>(ngy, (const T*)a.gy + r * a.ldgy, d, lane);
        if constexpr (GATE == ROW_GATE) load_row<T, NV, LANES, WIDTH>(ngate, (const T*)a.gate + r * a.ldg, d, lane);
    };
    const int64_t turn = (int64_t)gridDim.x * R::ROWS;
    int64_t r0 = (int64_t)blockIdx.x * R::ROWS;
    fetch(r0);
    for (; r0 < a.rows; r0 += turn) {
        const bool live = r0 + slot < a.rows;
        const int64_t r = live ? r0 + slot : a.rows - 1;
        const float4 st = nst;
        const P gy = ngy, block = nb;
        if constexpr (GATE == ROW_GATE) gate = ngate;
        auto there = [&](int i, int e) { return live && (i * LANES + lane) * CE + e < d; };
        Regs<T, NV> h, t;
        float w[CE], g[CE];
        // y as forward had it before rounding: the statistics are of that one
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T, NV, LANES, WIDTH>(h.v[i], block, i, d, lane);
            unpack<T, NV, LANES, WIDTH>(w, wpost, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) h.v[i][e] = (h.v[i][e] - st.x) * st.y * w[e];
            if constexpr (GATE != NO_GATE) {
                unpack<T, NV, LANES, WIDTH>(g, gate, i, d, lane);
#pragma unroll
                for (int e = 0; e < CE; ++e) h.v[i][e] *= g[e];
            }
            unpack<T, NV, LANES, WIDTH>(w, nx, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) h.v[i][e] = fmaf(a.scale, w[e], h.v[i][e]);
            unpack<T, NV, LANES, WIDTH>(g, ngn, i, d, lane, live && a.gn);
            unpack<T, NV, LANES, WIDTH>(w, wpre, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) {
                h.v[i][e] = there(i, e) ? (h.v[i][e] - st.z) * st.w : 0.0f;
                spre.v[i][e] = fmaf(g[e], h.v[i][e], spre.v[i][e]);
                t.v[i][e] = g[e] * w[e];
            }
        }
        if (r0 + turn < a.rows) fetch(r0 + turn);
        norm_back<T, NV, LANES>(t, h, d, a.layer, st.w, scratch);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T, NV, LANES, WIDTH>(g, gy, i, d, lane, live && a.gy);
#pragma unroll
            for (int e = 0; e < CE; ++e) {
                t.v[i][e] += g[e];
                h.v[i][e] = a.scale * t.v[i][e];
            }
        }
        store_row<T, NV, LANES>((T*)a.dx + r * d, h, d, lane, live);
        Regs<T, NV> dg;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            unpack<T, NV, LANES, WIDTH>(h.v[i], block, i, d, lane);
            unpack<T, NV, LANES, WIDTH>(w, wpost, i, d, lane);
            if constexpr (GATE != NO_GATE) unpack<T, NV, LANES, WIDTH>(g, gate, i, d, lane);
#pragma unroll
            for (int e = 0; e < CE; ++e) {
                h.v[i][e] = there(i, e) ? (h.v[i][e] - st.x) * st.y : 0.0f;
                if constexpr (GATE != NO_GATE) {
                    dg.v[i][e] = t.v[i][e] * h.v[i][e] * w[e];
                    if (GATE == CHANNEL_GATE && live) sgate.v[i][e] += dg.v[i][e];
                    t.v[i][e] *= g[e];
                }
                if (live) spost.v[i][e] = fmaf(t.v[i][e], h.v[i][e], spost.v[i][e]);
                t.v[i][e] *= w[e];
            }
        }
        if constexpr (GATE == ROW_GATE) store_row<T, NV, LANES>((T*)a.dgate_rows + r * d, dg, d, lane, live);
        norm_back<T, NV, LANES>(t, h, d, a.layer, st.y, scratch);
        store_row<T, NV, LANES>((T*)a.dblock + r * d, t, d, lane, live);
    }
    // column sums of the workgroup: its row slots, added in order, then its row of `partial`
    auto put = [&](int which, const Regs<T, NV>& s) {
        float* out = a.partial + ((int64_t)blockIdx.x * 3 + which) * d;
        if constexpr (R::ROWS == 1) {
            FOR_ROW(i, e) { const int c = (i * LANES + lane) * CE + e; if (c < d) out[c] = s.v[i][e]; }
        } else {
            __syncthreads();
            FOR_ROW(i, e) columns[slot * (LANES * NV * CE) + (i * LANES + lane) * CE + e] = s.v[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < d; c += R::THREADS) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < R::ROWS; ++k) v += columns[k * (LANES * NV * CE) + c];
                out[c] = v;
            }
        }
    };
    put(0, spost);
    put(1, spre);
    if constexpr (GATE == CHANNEL_GATE) put(2, sgate);
}

// dw_post, dw_pre, dgate: the partial rows added in a fixed order.  64 columns per workgroup, every 16th row per wave.
template <typename T>
__global__ __launch_bounds__(1024) void sum_columns_kernel(const float* __restrict__ partial, int blocks, int32_t d, T* __restrict__ o0, T* __restrict__ o1, T* __restrict__ o2) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int which = blockIdx.y, c = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < d)
#pragma unroll 8
        for (int b = wave; b < blocks; b += 16) s += partial[((int64_t)b * 3 + which) * d + c];
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < d) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += part[w][lane];
        T* o = which == 0 ? o0 : which == 1 ? o1 : o2;
        o[c] = from_f32<T>(s);
    }
}

// partial rows of backward: two workgroups of 512 threads or four of 256 on each of 256 CUs
constexpr int max_blocks(int32_t d) { return d <= 1024 ? 1024 : 512; }

// Threads per row and chunks per thread by width
template <typename T, class F> hipError_t by_width(int32_t d, F&& f) {
    const int chunks = (d + Chunk<T>::n - 1) / Chunk<T>::n;
    const bool whole = d % Chunk<T>::n == 0;
#define MARL_ROW(NV, LANES)                                                                                                          \
    return whole ? f(std::integral_constant<int, NV>{}, std::integral_constant<int, LANES>{}, std::integral_constant<int, WHOLE>{})  \
                 : f(std::integral_constant<int, NV>{}, std::integral_constant<int, LANES>{}, std::integral_constant<int, RAGGED>{})
    if (d < Chunk<T>::n) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{}, std::integral_constant<int, TINY>{});
    if (chunks <= 16) MARL_ROW(1, 16);
    if (chunks <= 32) MARL_ROW(1, 32);
    if (chunks <= 64) MARL_ROW(1, 64);
    if (chunks <= 128) MARL_ROW(1, 128);
    if (chunks <= 256) MARL_ROW(1, 256);
    if (chunks <= 512) MARL_ROW(1, 512);
    if (chunks <= 1024) MARL_ROW(2, 512);
    if (chunks <= 2048) MARL_ROW(2, 1024);
    if constexpr (Chunk<T>::n == 4) { if (chunks <= 4096) MARL_ROW(4, 1024); }
#undef MARL_ROW
    return hipErrorInvalidValue;
}

int done(hipError_t err) {
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

template <typename T> int forward(const NormArgs& a, hipStream_t stream) {
    return done(by_width<T>(a.d, [&](auto nv, auto lanes, auto width) {
        constexpr int NV = decltype(nv)::value, LANES = decltype(lanes)::value, WIDTH = decltype(width)::value;
        using R = Row<LANES>;
        const int64_t blocks = (a.rows + R::ROWS - 1) / R::ROWS, most = 256 * (2048 / R::THREADS);      // as many as the chip holds
        hipLaunchKernelGGL((residual_norm_kernel<T, NV, LANES, WIDTH>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(R::THREADS), 0, stream, a);
        return hipGetLastError();
    }));
}

template <typename T> int backward(const NormArgs& a, void* dw_post, void* dw_pre, void* dgate, hipStream_t stream) {
    int blocks = 0;
    hipError_t err = by_width<T>(a.d, [&](auto nv, auto lanes, auto width) {
        constexpr int NV = decltype(nv)::value, LANES = decltype(lanes)::value, WIDTH = decltype(width)::value;
        using R = Row<LANES>;
        // four turns or more a workgroup, so that adding the partial rows stays cheap, but one for every CU if there are rows
        const int64_t turns = (a.rows + R::ROWS - 1) / R::ROWS, want = turns / 4 > 256 ? turns / 4 : turns < 256 ? turns : 256;
        blocks = (int)(want < max_blocks(a.d) ? want : max_blocks(a.d));
        auto* kernel = a.gate_kind == NO_GATE        ? residual_norm_backward_kernel<T, NV, LANES, WIDTH, NO_GATE>
                       : a.gate_kind == CHANNEL_GATE ? residual_norm_backward_kernel<T, NV, LANES, WIDTH, CHANNEL_GATE>
                                                     : residual_norm_backward_kernel<T, NV, LANES, WIDTH, ROW_GATE>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(R::THREADS), 0, stream, a);
        return hipGetLastError();
    });
    if (err == hipSuccess) {
        hipLaunchKernelGGL(sum_columns_kernel<T>, dim3((a.d + 63) / 64, a.gate_kind == CHANNEL_GATE ? 3 : 2), dim3(1024), 0, stream, a.partial, blocks, a.d,
                           (T*)dw_post, (T*)dw_pre, (T*)dgate);
        err = hipGetLastError();
    }
    return done(err);
}

int check_sizes(int32_t dtype, int32_t kind, int64_t rows, int32_t d) {
    if (rows < 1 || d < 1 || dtype < MARL_F32 || dtype > MARL_F16 || kind < MARL_NORM_RMS || kind > MARL_NORM_LAYER) return MARL_EINVAL;
    if (d > MARL_MAX_NORM_WIDTH || rows > (1ll << 40)) return MARL_EUNSUPPORTED;
    return MARL_OK;
}

}  // namespace

extern "C" {

int marl_residual_norm(int32_t dtype, int32_t kind, int64_t rows, int32_t d, const void* x, int64_t ldx, const void* block, int64_t ld_block,
                       const void* w_post, const void* w_pre, const void* gate, int64_t ld_gate, float scale, float eps, void* y, void* n,
                       float* stats, void* stream) {
    const int rc = check_sizes(dtype, kind, rows, d);
    if (rc != MARL_OK) return rc;
    if (!x || !block || !w_post || !w_pre || !y || !n || !(eps >= 0.0f) || ((uintptr_t)stats & 15)) return MARL_EINVAL;
    if (rows > 1 && (ldx < d || ld_block < d || (gate && ld_gate != 0 && ld_gate < d))) return MARL_EINVAL;
    NormArgs a = {};
    a.x = x; a.block = block; a.w_post = w_post; a.w_pre = w_pre; a.gate = gate;
    a.ldx = ldx; a.ldb = ld_block; a.ldg = ld_gate;
    a.y = y; a.n = n; a.stats = stats; a.rows = rows; a.d = d;
    a.layer = kind == MARL_NORM_LAYER;
    a.gate_kind = !gate ? NO_GATE : ld_gate == 0 ? CHANNEL_GATE : ROW_GATE;
    a.scale = scale; a.eps = eps;
    return MARL_BY_TYPE(dtype, forward, a, (hipStream_t)stream);
}

size_t marl_residual_norm_workspace_bytes(int32_t d) {
    return d < 1 || d > MARL_MAX_NORM_WIDTH ? 0 : (size_t)max_blocks(d) * 3 * d * sizeof(float);
}

int marl_residual_norm_backward(int32_t dtype, int32_t kind, int64_t rows, int32_t d, const void* x, const void* block, int64_t ld_block,
                                const void* w_post, const void* w_pre, const void* gate, int64_t ld_gate, const float* stats, const void* gy,
                                int64_t ld_gy, const void* gn, int64_t ld_gn, float scale, void* dx, void* dblock, void* dw_post,
                                void* dw_pre, void* dgate, void* workspace, void* stream) {
    const int rc = check_sizes(dtype, kind, rows, d);
    if (rc != MARL_OK) return rc;
    if (!x || !block || !w_post || !w_pre || !stats || !dx || !dblock || !dw_post || !dw_pre || !workspace || (gate == nullptr) != (dgate == nullptr) ||
        ((uintptr_t)stats & 15) || ((uintptr_t)workspace & 15)) return MARL_EINVAL;
    if (rows > 1 && (ld_block < d || (gy && ld_gy < d) || (gn && ld_gn < d) || (gate && ld_gate != 0 && ld_gate < d))) return MARL_EINVAL;
    NormArgs a = {};
    a.block = block; a.w_post = w_post; a.w_pre = w_pre; a.gate = gate;
    a.x = x; a.ldx = d; a.ldb = ld_block; a.ldg = ld_gate;
    a.stats = const_cast<float*>(stats);
    a.gy = gy; a.gn = gn; a.ldgy = ld_gy; a.ldgn = ld_gn;
    a.dx = dx; a.dblock = dblock; a.dgate_rows = dgate; a.partial = (float*)workspace;
    a.rows = rows; a.d = d;
    a.layer = kind == MARL_NORM_LAYER;
    a.gate_kind = !gate ? NO_GATE : ld_gate == 0 ? CHANNEL_GATE : ROW_GATE;
    a.scale = scale;
    return MARL_BY_TYPE(dtype, backward, a, dw_post, dw_pre, a.gate_kind == CHANNEL_GATE ? dgate : nullptr, (hipStream_t)stream);
}

}  // extern "C"
