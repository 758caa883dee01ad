// Gated projections  y = act(a) * b,  a = x Wg^T, b = x Wu^T  (x [T, d], Wg and Wu [h, d]) and their gradients
//     da = gy p,  db = gy f,  f = act(a),  p = b act'(a),  dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x.
// All five contractions are one tiled product on the matrix cores, C[m][n] = sum_k A(m, k) B(n, k), in three settings:
//     FWD   A = x (k contiguous), B = rows of Wg and Wu in alternating groups of 32, so that a lane holds a and b of the
//           same (t, j) and the activation and the product happen in its registers
//     DX    A = [da | db] (k contiguous, 2h long), B = Wg then Wu with k along their rows
//     DW    A = [da | db]^T, B = x^T, both with k along their rows; the 2h rows of C are dWg then dWu
// Operands travel global -> LDS in 16-byte chunks (direct loads where every chunk is aligned and whole, through registers
// otherwise), two buffers of 128 bytes of k per row.  Tiles with k along the row are read back with ds_read_b128, tiles
// with k across the rows with ds_read_b64_tr_b16 (a 4 x 16 transpose in the read; float32 reads its single elements), so
// no transposed copy of a weight or a gradient is ever made.  Chunk positions are permuted within a row (tile_* below) so
// that the lanes of one LDS access fall on different banks.
// 16-bit types: v_mfma_f32_32x32x16 with float32 accumulators; float32: v_mfma_f32_32x32x2.  da and db are rounded to
// the element type, once, because they are matrix operands; f and p are kept in it between forward and backward (T h
// elements each, against 4 T d h operations for computing a and b again).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "marl_env.h"
#include "marl_net.h"
#include "marl_types.h"

extern "C" __attribute__((visibility("hidden"))) void marl_note_hip_error(int err);     // marl_env.hip

namespace {

using namespace marl_types;
using marl_net::floatx16;

enum Mode { FWD, DX, DW };
constexpr int ROW_BYTES = 128;               // bytes of k per tile row and step

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <typename T> struct Frag { typedef short8v type; };                // 8 elements of k per lane, two halves: 16
template <> struct Frag<float> { typedef floatx4 type; };                   // 4 elements of k per lane, two halves: 8

__device__ __forceinline__ floatx16 mma(bf16, short8v a, short8v b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(f16, short8v a, short8v b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(float, floatx4 a, floatx4 b, floatx16 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

// -- activations -----------------------------------------------------------------------------------------------------
template <bool FAST> __device__ __forceinline__ float exp_of(float x) { return FAST ? __expf(x) : expf(x); }

// f = act(a) and its derivative; FAST: the hardware exponential, whose error (a few 2^-22) is far below a 16-bit step
template <int ACT, bool FAST> __device__ __forceinline__ void act_both(float a, float& f, float& df) {
    if constexpr (ACT == MARL_ACT_RELU) {
        f = a > 0.0f ? a : (a != a ? a : 0.0f);
        df = a > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == MARL_ACT_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * a);
        f = a * cdf;
        df = cdf + a * 0.39894228040143268f * exp_of<FAST>(-0.5f * a * a);
    } else {
        const float s = 1.0f / (1.0f + exp_of<FAST>(-a));
        if constexpr (ACT == MARL_ACT_SIGMOID) { f = s; df = s * (1.0f - s); }
        else { f = a * s; df = s * (1.0f + a * (1.0f - s)); }
    }
}
template <class F> __device__ __forceinline__ void by_act(int act, F&& f) {
    switch (act) {
        case MARL_ACT_SILU: f(std::integral_constant<int, MARL_ACT_SILU>{}); break;
        case MARL_ACT_GELU: f(std::integral_constant<int, MARL_ACT_GELU>{}); break;
        case MARL_ACT_RELU: f(std::integral_constant<int, MARL_ACT_RELU>{}); break;
        default: f(std::integral_constant<int, MARL_ACT_SIGMOID>{}); break;
    }
}

// -- tiles -----------------------------------------------------------------------------------------------------------
struct Operand {
    const void *p0, *p1;      // p1: the second weight (FWD: odd groups of 32 rows, DX: k >= h)
    int64_t ld0, ld1;
};
struct ProductArgs {
    Operand A, B;
    int64_t M, N, K;          // FWD: M = T, N = h, K = d.  DX: T, d, 2h.  DW: 2h, d, T.
    int64_t h;
    int64_t k_chunk;          // k range of one z slice, a multiple of the step
    void *out0, *out1;        // FWD: y; DX: dx; DW: dWg, dWu
    void *save_f, *save_p;    // FWD: NULL, or what backward needs
    float* partial;           // [slices][M][N] when the k range is split
    int act;
    int tiles_m, tiles_n;
};

template <typename T, int ACT> __device__ __forceinline__ void gate_out(const ProductArgs& args, int64_t at, float a, float b) {
    float f, df;
    act_both<ACT, sizeof(T) == 2>(a, f, df);
    ((T*)args.out0)[at] = from_f32<T>(f * b);
    if (args.save_f) {
        ((T*)args.save_f)[at] = from_f32<T>(f);
        ((T*)args.save_p)[at] = from_f32<T>(b * df);
    }
}

// position of chunk c in row r of a tile with k along the row (8 chunks a row)
__device__ __forceinline__ int tile_k_along(int r, int c) { return c ^ (r & 7); }
// position of chunk c in k-row kr of a tile with k across the rows.  16-bit: pairs of chunks (the 16 elements one
// transposing read takes from a row) are permuted by the four rows and the row octet that one access covers; float32:
// the two half waves read rows four apart, which go to different 128-byte halves.
template <typename T> __device__ __forceinline__ int tile_k_across(int kr, int c) {
    if constexpr (sizeof(T) == 2) return c ^ (((kr & 3) | (((kr >> 3) & 1) << 2)) << 1);
    else return c ^ (((kr >> 2) & 1) << 3);
}

typedef __attribute__((address_space(3))) char lds_char;

// One operand's tile: ROWS rows (m or n) by ROW_BYTES of k.  ACROSS: k runs across the rows of memory.
template <typename T, int MODE, bool IS_B, int ROWS, int THREADS>
struct Tile {
    static constexpr int CE = Chunk<T>::n;
    static constexpr int BK = ROW_BYTES / (int)sizeof(T);
    static constexpr bool ACROSS = MODE == DW || (MODE == DX && IS_B);
    static constexpr int CHUNKS = ROWS * 8;
    static constexpr int PER = CHUNKS / THREADS;
    static constexpr int CPR = ACROSS ? ROWS / CE : 8;         // chunks of a memory row
    static_assert(CHUNKS % THREADS == 0, "whole chunks per thread");

    // chunk q of the tile: (row of memory, first element in it, both inside the tile)
    static __device__ __forceinline__ void place(int q, int& r, int& e) {
        r = q / CPR;
        const int pos = q % CPR;
        e = (ACROSS ? tile_k_across<T>(r, pos) : tile_k_along(r, pos)) * CE;
    }
    // address of memory row `r` of the tile that starts at (row0, k0); FWD's B: groups of 32 rows, gate and up in turn
    static __device__ __forceinline__ const T* row_ptr(const ProductArgs& a, int64_t row0, int64_t k0, int r, int64_t& row, int64_t rows) {
        const Operand& o = IS_B ? a.B : a.A;
        if constexpr (ACROSS) {
            row = k0 + r;
            if constexpr (MODE == DX) {
                const bool second = row >= a.h;
                return (const T*)(second ? o.p1 : o.p0) + (second ? row - a.h : row) * (second ? o.ld1 : o.ld0);
            }
            return (const T*)o.p0 + row * o.ld0;
        } else if constexpr (MODE == FWD && IS_B) {
            row = row0 / 2 + (r / 64) * 32 + (r & 31);
            const bool up = (r & 32) != 0;
            const int64_t rr = row < rows ? row : rows - 1;
            return (const T*)(up ? o.p1 : o.p0) + rr * (up ? o.ld1 : o.ld0);
        } else {
            row = row0 + r;
            const int64_t rr = row < rows ? row : rows - 1;
            return (const T*)o.p0 + rr * o.ld0;
        }
    }
    // The thread's chunks at k = 0, found once: a step then adds one offset to all of them.  DX's B reads the second
    // weight from k = h on: its chunks at k = h.
    struct Pointers {
        const T* at[PER];
        const T* at2[MODE == DX && IS_B ? PER : 1];
    };
    static __device__ __forceinline__ void pointers(const ProductArgs& a, int64_t row0, int64_t rows, Pointers& p) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, e;
            place(i * THREADS + (int)threadIdx.x, r, e);
            if constexpr (ACROSS) {       // columns beyond the edge repeat the last chunk (their results are never stored)
                const int64_t col = row0 + e < rows ? row0 + e : rows - CE;
                const Operand& o = IS_B ? a.B : a.A;
                p.at[i] = (const T*)o.p0 + r * o.ld0 + col;
                if constexpr (MODE == DX) p.at2[i] = (const T*)o.p1 + r * o.ld1 + col;
            } else {                      // rows beyond the edge repeat the last one
                int64_t row;
                p.at[i] = row_ptr(a, row0, 0, r, row, rows) + e;
            }
        }
    }
    // direct global -> LDS: every k of the step exists (DX: on one side of h), chunks are aligned and whole
    static __device__ __forceinline__ void load_direct(const ProductArgs& a, const Pointers& p, int64_t k0, char* lds) {
        const Operand& o = IS_B ? a.B : a.A;
        const bool second = MODE == DX && IS_B && k0 >= a.h;
        const int64_t step = !ACROSS ? k0 : second ? (k0 - a.h) * o.ld1 : k0 * o.ld0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const T* src = p.at[i];
            if constexpr (MODE == DX && IS_B) src = second ? p.at2[i] : src;
            char* dst = lds + (size_t)(i * THREADS + (threadIdx.x & ~63)) * 16;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + step),
                                             (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
        }
    }
    // through registers: any alignment, zeros beyond the edges
    static __device__ __forceinline__ void load_masked(const ProductArgs& a, int64_t row0, int64_t rows, int64_t k0, int64_t k_end, Vec<T> (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, e;
            place(i * THREADS + (int)threadIdx.x, r, e);
            int64_t row, left;
            if constexpr (ACROSS) {
                left = k0 + r < k_end ? rows - (row0 + e) : 0;
                const T* p = row_ptr(a, row0, left > 0 ? k0 : 0, left > 0 ? r : 0, row, rows) + row0 + e;
                v[i] = load_part(p, left);
            } else {
                left = k_end - (k0 + e);
                v[i] = load_part(row_ptr(a, row0, k0, r, row, rows) + k0 + e, left);
            }
        }
    }
    static __device__ __forceinline__ void store_lds(char* lds, const Vec<T> (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; ++i) *(Vec<T>*)(lds + (size_t)(i * THREADS + threadIdx.x) * 16) = v[i];
    }
    // the lane's operand of the 32 rows from `base` on for k step ks (16 elements of k, float32: 8)
    static __device__ __forceinline__ typename Frag<T>::type frag(const char* lds, int base, int ks, int lane) {
        if constexpr (!ACROSS) {
            const int r = base + (lane & 31);
            return *(const typename Frag<T>::type*)(lds + r * ROW_BYTES + tile_k_along(r, 2 * ks + (lane >> 5)) * 16);
        } else if constexpr (sizeof(T) == 2) {
            const int g = lane >> 4, i = lane & 15;
            const int c = base / 8 + 2 * (g & 1) + ((i >> 1) & 1);
            short8v out;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int kr = 16 * ks + 8 * (g >> 1) + 4 * half + (i >> 2);
                const char* p = lds + kr * (ROWS * 2) + tile_k_across<T>(kr, c) * 16 + (i & 1) * 8;
                const short4v t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
#pragma unroll
                for (int s = 0; s < 4; ++s) out[4 * half + s] = t[s];
            }
            return out;
        } else {
            const int m = base + (lane & 31);
            floatx4 out;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int kr = 8 * ks + 4 * (lane >> 5) + s;
                out[s] = *(const float*)(lds + kr * (ROWS * 4) + tile_k_across<T>(kr, m >> 2) * 16 + (m & 3) * 4);
            }
            return out;
        }
    }
};

// Tile of C that a block computes: consecutive blocks go to the eight XCDs in turn, so block ids are first regrouped
// (ids of one XCD side by side), then walked in bands of eight row tiles: what an XCD works on at a time shares its
// operand rows in that XCD's L2.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, per = total / 8, rest = total % 8;
    const int xcd = id % 8, slot = id / 8;
    const int t = xcd * per + (xcd < rest ? xcd : rest) + slot;
    constexpr int BAND = 8;
    const int band = t / (BAND * tiles_n), first = band * BAND;
    const int height = tiles_m - first < BAND ? tiles_m - first : BAND;
    const int in = t - band * BAND * tiles_n;
    tm = first + in % height;
    tn = in / height;
}

template <typename T, int MODE, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(const ProductArgs args) {
    constexpr int THREADS = WM * WN * 64;
    using TA = Tile<T, MODE, false, BM, THREADS>;
    using TB = Tile<T, MODE, true, BN, THREADS>;
    constexpr int BK = TA::BK, KSTEPS = BK / (sizeof(T) == 2 ? 16 : 8);
    constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
    constexpr int A_BYTES = BM * ROW_BYTES, B_BYTES = BN * ROW_BYTES, BUF = A_BYTES + B_BYTES;
    static_assert(MODE != FWD || NI == 2, "one gate and one up group per wave");
    extern __shared__ __align__(128) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    int tm, tn;
    tile_of(blockIdx.x, args.tiles_m, args.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;              // FWD: n0 counts gate and up rows
    const int64_t k_begin = (int64_t)blockIdx.y * args.k_chunk;
    const int64_t k_end = k_begin + args.k_chunk < args.K ? k_begin + args.k_chunk : args.K;
    const int steps = (int)((k_end - k_begin + BK - 1) / BK);
    floatx16 acc[MI][NI] = {};
    Vec<T> va[TA::PER], vb[TB::PER];
    typename TA::Pointers pa;
    typename TB::Pointers pb;
    if (DIRECT) { TA::pointers(args, m0, args.M, pa); TB::pointers(args, n0, args.N, pb); }

    // Step s into `buf`: direct loads, or (a ragged step; every step if !DIRECT) into registers, which commit() stores.
    auto fetch = [&](int s, char* buf) {
        const int64_t k0 = k_begin + (int64_t)s * BK;
        if (DIRECT && k0 + BK <= k_end && (MODE != DX || k0 + BK <= args.h || k0 >= args.h)) {
            TA::load_direct(args, pa, k0, buf);
            TB::load_direct(args, pb, k0, buf + A_BYTES);
        } else {
            TA::load_masked(args, m0, args.M, k0, k_end, va);
            TB::load_masked(args, n0, args.N, k0, k_end, vb);
            if (DIRECT) { TA::store_lds(buf, va); TB::store_lds(buf + A_BYTES, vb); }
        }
    };
    auto commit = [&](char* buf) {
        if (!DIRECT) { TA::store_lds(buf, va); TB::store_lds(buf + A_BYTES, vb); }
    };
    typename Frag<T>::type fa[2][MI], fb[2][NI];
    auto read = [&](const char* buf, int ks, int to) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[to][i] = TA::frag(buf, wm * (BM / WM) + 32 * i, ks, lane);
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[to][j] = TB::frag(buf + A_BYTES, wn * (BN / WN) + 32 * j, ks, lane);
    };
    auto multiply = [&](int from) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mma(T(), fa[from][i], fb[from][j], acc[i][j]);
    };
    // Operands are read one k step ahead of their use, and the barrier between two buffers stands before the last
    // k step's products, which cover the first reads of the new buffer.
    fetch(0, lds);
    commit(lds);
    __syncthreads();
    read(lds, 0, 0);
    for (int s = 0; s < steps; ++s) {
        char* cur = lds + (s & 1) * BUF;
        char* nxt = lds + ((s + 1) & 1) * BUF;
        if (s + 1 < steps) fetch(s + 1, nxt);
#pragma unroll
        for (int ks = 0; ks + 1 < KSTEPS; ++ks) {
            read(cur, ks + 1, (ks + 1) & 1);
            multiply(ks & 1);
        }
        if (s + 1 < steps) commit(nxt);
        __syncthreads();
        if (s + 1 < steps) read(nxt, 0, 0);
        multiply((KSTEPS - 1) & 1);
    }
    // register v of a lane: row 8 (v / 4) + 4 (lane / 32) + v % 4, column lane % 32
    const int hl = lane >> 5, col = lane & 31;
    if constexpr (MODE == FWD) {
        const int64_t n = n0 / 2 + wn * 32 + col;
        if (n >= args.N) return;
        by_act(args.act, [&](auto kind) {
            constexpr int ACT = decltype(kind)::value;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int64_t m = m0 + wm * (BM / WM) + 32 * i + 8 * (v / 4) + 4 * hl + v % 4;
                    if (m >= args.M) continue;
                    gate_out<T, ACT>(args, m * args.N + n, acc[i][0][v], acc[i][1][v]);
                }
        });
    } else {
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int64_t n = n0 + wn * (BN / WN) + 32 * j + col;
            if (n >= args.N) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int64_t m = m0 + wm * (BM / WM) + 32 * i + 8 * (v / 4) + 4 * hl + v % 4;
                    if (m >= args.M) continue;
                    if (args.partial) args.partial[((int64_t)blockIdx.y * args.M + m) * args.N + n] = acc[i][j][v];
                    else if (MODE == DW && m >= args.h) ((T*)args.out1)[(m - args.h) * args.N + n] = from_f32<T>(acc[i][j][v]);
                    else ((T*)args.out0)[m * args.N + n] = from_f32<T>(acc[i][j][v]);
                }
        }
    }
}

// Sum of the k slices, rounded once.  `first` elements go to out0, the rest to out1.
template <typename T>
__global__ __launch_bounds__(256) void sum_slices_kernel(const float* __restrict__ partial, int slices, int64_t n, int64_t first, T* __restrict__ out0, T* __restrict__ out1) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int z = 0; z < slices; ++z) s += partial[z * n + i];
        if (i < first) out0[i] = from_f32<T>(s);
        else out1[i - first] = from_f32<T>(s);
    }
}

// Few rows (T <= 32 MT): the weights are read once and nothing else counts.  A block owns 32 columns j (rows of both
// weights), its eight waves split d; a lane reads 64 consecutive bytes of one weight row and of one row of x, straight
// into matrix operands (the order of k inside a run is the same for both, so it needs no shuffle).  The eight partial
// sums meet in LDS.
template <typename T, int MT>
__global__ __launch_bounds__(512) void gated_few_rows_kernel(const ProductArgs args) {
    constexpr int CE = Chunk<T>::n, RUN = 8 * CE, WAVES = 8;                // 4 chunks per half wave
    extern __shared__ __align__(128) char lds[];
    float* part = (float*)lds;                                              // [WAVES][MT][2][16][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane >> 5, r = lane & 31;
    const int64_t j = (int64_t)blockIdx.x * 32 + r, d = args.K;
    const int64_t jj = j < args.N ? j : args.N - 1;
    const T* wg = (const T*)args.B.p0 + jj * args.B.ld0;
    const T* wu = (const T*)args.B.p1 + jj * args.B.ld1;
    const T* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t t = 32 * i + r < args.M ? 32 * i + r : args.M - 1;
        x[i] = (const T*)args.A.p0 + t * args.A.ld0;
    }
    floatx16 acc[MT][2] = {};
    for (int64_t k0 = (int64_t)wave * RUN; k0 < d; k0 += WAVES * RUN) {
        const int64_t k = k0 + hl * 4 * CE;
        Vec<T> g[4], u[4], xv[MT][4];
        if (k0 + RUN <= d) {
#pragma unroll
            for (int c = 0; c < 4; ++c) { g[c] = load_chunk(wg + k + c * CE); u[c] = load_chunk(wu + k + c * CE); }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) xv[i][c] = load_chunk(x[i] + k + c * CE);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int64_t left = d - (k + c * CE);
                g[c] = load_part(wg + k + c * CE, left);
                u[c] = load_part(wu + k + c * CE, left);
#pragma unroll
                for (int i = 0; i < MT; ++i) xv[i][c] = load_part(x[i] + k + c * CE, left);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                using F = typename Frag<T>::type;
                acc[i][0] = mma(T(), __builtin_bit_cast(F, xv[i][c]), __builtin_bit_cast(F, g[c]), acc[i][0]);
                acc[i][1] = mma(T(), __builtin_bit_cast(F, xv[i][c]), __builtin_bit_cast(F, u[c]), acc[i][1]);
            }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int v = 0; v < 16; ++v) part[(((wave * MT + i) * 2 + w) * 16 + v) * 64 + lane] = acc[i][w][v];
    __syncthreads();
    if (j >= args.N) return;
    by_act(args.act, [&](auto kind) {
        constexpr int ACT = decltype(kind)::value;
        for (int iv = wave; iv < 16 * MT; iv += WAVES) {
            const int i = iv / 16, v = iv % 16;
            const int64_t t = 32 * i + 8 * (v / 4) + 4 * hl + v % 4;
            if (t >= args.M) continue;
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                a += part[(((w * MT + i) * 2 + 0) * 16 + v) * 64 + lane];
                b += part[(((w * MT + i) * 2 + 1) * 16 + v) * 64 + lane];
            }
            gate_out<T, ACT>(args, t * args.N + j, a, b);
        }
    });
}

// [da | db] = [gy p | gy f] of every row: bandwidth (three reads, two writes of T h)
template <typename T>
__global__ __launch_bounds__(256) void gated_da_db_kernel(const T* __restrict__ f, const T* __restrict__ p, const T* __restrict__ gy, int64_t ldgy,
                                                           T* __restrict__ dab, int64_t rows, int64_t h) {
    constexpr int CE = Chunk<T>::n;
    const int64_t per = (h + CE - 1) / CE;
    for (int64_t t = blockIdx.y; t < rows; t += gridDim.y)
        for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < per; q += (int64_t)gridDim.x * 256) {
            const int64_t c = q * CE, left = h - c;
            const Vec<T> vf = load_part(f + t * h + c, left), vp = load_part(p + t * h + c, left), vg = load_part(gy + t * ldgy + c, left);
            Vec<T> da, db;
#pragma unroll
            for (int i = 0; i < CE; ++i) {
                const float g = to_f32(vg.e[i]);
                da.e[i] = from_f32<T>(g * to_f32(vp.e[i]));
                db.e[i] = from_f32<T>(g * to_f32(vf.e[i]));
            }
            store_part(dab + t * 2 * h + c, da, left);
            store_part(dab + t * 2 * h + h + c, db, left);
        }
}

// -- host ------------------------------------------------------------------------------------------------------------
template <typename T> bool whole(const void* p, int64_t ld, int64_t n) {
    return ((uintptr_t)p & 15) == 0 && ld % Chunk<T>::n == 0 && n % Chunk<T>::n == 0;
}

struct Plan { bool big; int slices; int64_t k_chunk; };

// Tile and split of one product.  256 x 256 tiles (one block of eight waves per CU) where they fill the chip, else
// 128 x 128 (two blocks per CU); if those do not fill it either, the k range is cut into slices of at least eight steps.
template <typename T> Plan plan_of(int mode, int64_t M, int64_t N, int64_t K) {
    const int cus = marl_net::device_cus(256);
    const int64_t bk = ROW_BYTES / sizeof(T);
    Plan p;
    auto tiles = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
    const int64_t steps = K > 0 ? (K + bk - 1) / bk : 1;
    p.big = tiles(256) >= cus * 3 / 4;
    p.slices = 1;
    if (mode != FWD && !p.big) {
        const int64_t want = 2 * cus / tiles(128);
        p.slices = (int)(want < 1 ? 1 : want < steps / 8 ? want : steps / 8 < 1 ? 1 : steps / 8);
    }
    p.k_chunk = ((steps + p.slices - 1) / p.slices) * bk;
    p.slices = (int)((steps * bk + p.k_chunk - 1) / p.k_chunk);
    return p;
}

template <typename T, int MODE, int BM, int WM, int WN, bool DIRECT>
hipError_t launch_tiles(ProductArgs& a, int64_t n_virtual, const Plan& p, hipStream_t stream) {
    static bool attr_set[marl_net::kMaxDevices];
    auto* kernel = product_kernel<T, MODE, BM, BM, WM, WN, DIRECT>;
    const size_t bytes = (size_t)4 * BM * ROW_BYTES;
    hipError_t err = marl_net::allow_dynamic_lds((const void*)kernel, bytes, attr_set);
    if (err != hipSuccess) return err;
    a.tiles_m = (int)((a.M + BM - 1) / BM);
    a.tiles_n = (int)((n_virtual + BM - 1) / BM);
    a.k_chunk = p.k_chunk;
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n, p.slices), dim3(WM * WN * 64), bytes, stream, a);
    return hipGetLastError();
}

template <typename T, int MODE>
hipError_t launch_product(ProductArgs& a, float* partial, hipStream_t stream) {
    const int64_t n_virtual = MODE == FWD ? ((a.N + 31) / 32) * 64 : a.N;       // FWD: gate and up in groups of 32
    const Plan p = plan_of<T>(MODE, a.M, n_virtual, a.K);
    a.partial = p.slices > 1 ? partial : nullptr;
    // direct loads: whole aligned chunks in both operands.  k along the row: the ragged end goes through registers
    bool direct = MODE == DW ? whole<T>(a.A.p0, a.A.ld0, a.M) && whole<T>(a.B.p0, a.B.ld0, a.N)
                             : whole<T>(a.A.p0, a.A.ld0, 0) && whole<T>(a.B.p0, a.B.ld0, MODE == DX ? a.N : 0) &&
                                   whole<T>(a.B.p1, a.B.ld1, MODE == DX ? a.N : 0);
    hipError_t err;
    if (p.big) err = direct ? launch_tiles<T, MODE, 256, 2, 4, true>(a, n_virtual, p, stream) : launch_tiles<T, MODE, 256, 2, 4, false>(a, n_virtual, p, stream);
    else err = direct ? launch_tiles<T, MODE, 128, 2, 2, true>(a, n_virtual, p, stream) : launch_tiles<T, MODE, 128, 2, 2, false>(a, n_virtual, p, stream);
    if (err != hipSuccess || a.partial == nullptr) return err;
    const int64_t n = a.M * a.N;
    const int64_t first = MODE == DW ? a.h * a.N : n;
    const int64_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(sum_slices_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, partial, p.slices, n, first, (T*)a.out0, (T*)a.out1);
    return hipGetLastError();
}

template <typename T, int MT> hipError_t launch_few_rows(const ProductArgs& a, hipStream_t stream) {
    static bool attr_set[marl_net::kMaxDevices];
    const size_t bytes = (size_t)8 * MT * 2 * 16 * 64 * sizeof(float);
    hipError_t err = marl_net::allow_dynamic_lds((const void*)gated_few_rows_kernel<T, MT>, bytes, attr_set);
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL((gated_few_rows_kernel<T, MT>), dim3((unsigned)((a.N + 31) / 32)), dim3(512), bytes, stream, a);
    return hipGetLastError();
}

template <typename T> int forward(int act, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                  const void* wu, int64_t ldu, void* y, void* f, void* p, hipStream_t stream) {
    ProductArgs a = {};
    a.A = {x, nullptr, ldx, 0};
    a.B = {wg, wu, ldg, ldu};
    a.M = rows; a.N = h; a.K = d; a.h = h;
    a.out0 = y; a.save_f = f; a.save_p = p; a.act = act;
    hipError_t err = rows <= 32 ? launch_few_rows<T, 1>(a, stream) : rows <= 64 ? launch_few_rows<T, 2>(a, stream) : launch_product<T, FWD>(a, nullptr, stream);
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

int64_t round_256(int64_t n) { return (n + 255) / 256 * 256; }

template <typename T> size_t workspace(int64_t rows, int32_t d, int32_t h) {
    const Plan px = plan_of<T>(DX, rows, d, 2 * (int64_t)h), pw = plan_of<T>(DW, 2 * (int64_t)h, d, rows);
    const int64_t sx = px.slices > 1 ? px.slices * rows * d : 0, sw = pw.slices > 1 ? pw.slices * 2 * (int64_t)h * d : 0;
    return (size_t)(round_256(rows * 2 * h * (int64_t)sizeof(T)) + (sx > sw ? sx : sw) * (int64_t)sizeof(float));
}

template <typename T> int backward(int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                   const void* wu, int64_t ldu, const void* f, const void* p, const void* gy, int64_t ldgy, void* dx,
                                   void* dwg, void* dwu, void* ws, hipStream_t stream) {
    T* dab = (T*)ws;
    float* partial = (float*)((char*)ws + round_256(rows * 2 * h * (int64_t)sizeof(T)));
    const int64_t per = (h + Chunk<T>::n - 1) / Chunk<T>::n;
    hipLaunchKernelGGL(gated_da_db_kernel<T>, dim3((unsigned)((per + 255) / 256), (unsigned)(rows < 65535 ? rows : 65535)), dim3(256), 0, stream,
                       (const T*)f, (const T*)p, (const T*)gy, ldgy, dab, rows, (int64_t)h);
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && dx) {
        ProductArgs a = {};
        a.A = {dab, nullptr, 2 * (int64_t)h, 0};
        a.B = {wg, wu, ldg, ldu};
        a.M = rows; a.N = d; a.K = 2 * (int64_t)h; a.h = h; a.out0 = dx;
        err = launch_product<T, DX>(a, partial, stream);
    }
    if (err == hipSuccess && dwg) {
        ProductArgs a = {};
        a.A = {dab, nullptr, 2 * (int64_t)h, 0};
        a.B = {x, nullptr, ldx, 0};
        a.M = 2 * (int64_t)h; a.N = d; a.K = rows; a.h = h; a.out0 = dwg; a.out1 = dwu;
        err = launch_product<T, DW>(a, partial, stream);
    }
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

int check_sizes(int32_t dtype, int32_t act, int64_t rows, int32_t d, int32_t h) {
    if (rows < 1 || d < 1 || h < 1) return MARL_EINVAL;
    if (dtype < MARL_F32 || dtype > MARL_F16 || act < MARL_ACT_SILU || act > MARL_ACT_SIGMOID) return MARL_EINVAL;
    // tile and block counts stay below 2^31
    if (rows > (1ll << 31) - 256 || d > (1 << 24) || h > (1 << 24) || ((rows + 127) / 128) * (((int64_t)h + 31) / 32) > (1ll << 30) ||
        ((rows + 127) / 128) * (((int64_t)d + 31) / 32) > (1ll << 30)) return MARL_EUNSUPPORTED;
    return MARL_OK;
}

}  // namespace

extern "C" {

int marl_gated_forward(int32_t dtype, int32_t act, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* w_gate,
                       int64_t ld_gate, const void* w_up, int64_t ld_up, void* y, void* f, void* p, void* stream) {
    const int rc = check_sizes(dtype, act, rows, d, h);
    if (rc != MARL_OK) return rc;
    if (!x || !w_gate || !w_up || !y || (f == nullptr) != (p == nullptr)) return MARL_EINVAL;
    if (ldx < d && rows > 1) return MARL_EINVAL;
    if ((ld_gate < d || ld_up < d) && h > 1) return MARL_EINVAL;
    return MARL_BY_TYPE(dtype, forward, act, rows, d, h, x, ldx, w_gate, ld_gate, w_up, ld_up, y, f, p, (hipStream_t)stream);
}

size_t marl_gated_workspace_bytes(int32_t dtype, int64_t rows, int32_t d, int32_t h) {
    if (check_sizes(dtype, MARL_ACT_SILU, rows, d, h) != MARL_OK) return 0;
    return MARL_BY_TYPE(dtype, workspace, rows, d, h);
}

int marl_gated_backward(int32_t dtype, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* w_gate,
                        int64_t ld_gate, const void* w_up, int64_t ld_up, const void* f, const void* p, const void* gy, int64_t ld_gy,
                        void* dx, void* dw_gate, void* dw_up, void* workspace_, void* stream) {
    const int rc = check_sizes(dtype, MARL_ACT_SILU, rows, d, h);
    if (rc != MARL_OK) return rc;
    if (!x || !w_gate || !w_up || !f || !p || !gy || !workspace_ || ((uintptr_t)workspace_ & 15) || (dw_gate == nullptr) != (dw_up == nullptr)) return MARL_EINVAL;
    if ((ldx < d || ld_gy < h) && rows > 1) return MARL_EINVAL;
    if ((ld_gate < d || ld_up < d) && h > 1) return MARL_EINVAL;
    return MARL_BY_TYPE(dtype, backward, rows, d, h, x, ldx, w_gate, ld_gate, w_up, ld_up, f, p, gy, ld_gy, dx, dw_gate, dw_up, workspace_,
                        (hipStream_t)stream);
}

}  // extern "C"
