// Gated projections  y = act(a) * b,  a = x Wg^T, b = x Wu^T  (x [T, d], Wg and Wu [h, d]) and their gradients
//     da = gy p,  db = gy f,  f = act(a),  p = b act'(a),  dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x.
// All five contractions are one tiled product on the matrix cores, C[m][n] = sum_k A(m, k) B(n, k), in three settings:
//     FWD   A = x (k contiguous), B = rows of Wg and Wu in alternating groups of 32, so that a lane holds a and b of the
//           same (t, j) and the activation and the product happen in its registers
//     DX    A = [da | db] (k contiguous), B = Wg then Wu with k across their rows
//     DW    A = [da | db]^T, B = x^T, both with k across their rows; the 2h rows of C are dWg then dWu
// Operands travel global -> LDS in 16-byte chunks by direct loads (a ragged last step of k through registers) into a ring
// of five stages of 64 bytes of k per row: three stages are under way while one is multiplied, which covers the latency of
// a miss in L2 (with two stages of 128 bytes the loop waited for memory half of its time), and the fifth place lets a wave
// pass a barrier without waiting for its own LDS reads.  Operands whose rows are not
// aligned to chunks are first copied to rows that are.  Tiles with k along the row are read back with ds_read_b128, tiles
// with k across the rows with ds_read_b64_tr_b16 (a 4 x 16 transpose in the read; float32 reads its single elements), so
// no transposed copy of a weight or a gradient is ever made.  Chunk positions are permuted within a row (tile_* below) so
// that the lanes of one LDS access fall on different banks.
// 16-bit types: v_mfma_f32_32x32x16 with float32 accumulators; float32: v_mfma_f32_32x32x2.  da and db are rounded to
// the element type, once, because they are matrix operands.  f and p are kept between forward and backward in float32, T h
// elements each, against 4 T d h operations for computing a and b again: in 16 bits da and db would be rounded twice
// (gradients off by 0.0029 instead of 0.0023 in bf16), and p = b act'(a) may lie outside of float16 where y and the gradients
// do not.
// Bound by the matrix cores; FWD / DX / DW measured: T 8192, d 2048, h 8192, bf16: 636 / 462 / 469 us (865 / 1190 / 1172
// TFLOP/s; FWD without f and p 476 us: the rest is their stores, behind which a block's matrix cores idle); T 32768, d 128,
// h 512, float32: 103 / 79 / 77 us (83 / 109 / 112); T 1999, d 1000, h 2731, float16: 54 / 36 / 36 us (404 / 601 / 605), at
// d 1001 six copies of operands of 4.5 us each more in a step.  da and db are bandwidth: 156 us at the first sizes (6.0 TB/s).
// Few rows are bound by the weights' bytes: T 1, d 2048, h 8192, bf16: 14.0 us a call (4.8 TB/s).  Far from any bound: forward
// of more than 64 rows over narrow weights, whose few tiles each run all of k (T 128, d 4096, h 512: 33 us in bf16, 239 in
// float32, where 64 rows take 27 and 25).
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
constexpr int ROW_BYTES = 64;                // bytes of k per tile row and stage
constexpr int STAGES = 5, AHEAD = 3;         // places of the ring; stages under way while one is multiplied

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
    const void *p0, *p1;      // p1: the second weight (FWD: odd groups of 32 rows, DX: the second pass over k)
    int64_t ld0, ld1;
};
struct ProductArgs {
    Operand A, B;
    int64_t M, N, K;          // FWD: M = T, N = h, K = d.  DX: T, d, h, twice: for da and for db.  DW: 2 half, d, T.
    int64_t h, half;          // backward: db stands `half` columns behind da (h rounded up to whole chunks)
    int stages;               // stages of k in one slice
    void *out0, *out1;        // FWD: y; DX: dx; DW: dWg, dWu
    float *save_f, *save_p;   // FWD: NULL, or what backward needs
    float* partial;           // [slices][M][N] when the k range is split
    int act;
    int tiles_m, tiles_n;
};

template <int N> __device__ __forceinline__ void stream_floats(float* p, const float (&v)[N], int64_t left) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        const Part<float, 4> t = {{v[c], v[c + 1], v[c + 2], v[c + 3]}};
        if (left > c) stream_part(p + c, t, left - c);
    }
}
// y, and f and p for backward, of `left` (at most W) neighbouring columns from their a and b; stored past the caches,
// which hold the operands (T 32768, d 128, h 512, float32: 115 -> 103 us)
// W columns: a chunk, or four.
template <typename T, int ACT, int W> __device__ __forceinline__ void gate_out(const ProductArgs& args, int64_t at, const float* a, const float* b, int64_t left) {
    Part<T, W> y;
    float f[W], p[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
        float df;
        act_both<ACT, sizeof(T) == 2>(a[e], f[e], df);
        y.e[e] = from_f32<T>(f[e] * b[e]);
        p[e] = b[e] * df;
    }
    stream_part((T*)args.out0 + at, y, left);
    if (args.save_f) {
        stream_floats(args.save_f + at, f, left);
        stream_floats(args.save_p + at, p, left);
    }
}

// position of chunk c in row r of a tile with k along the row (4 chunks a row): sixteen consecutive rows, read at one
// chunk, cover all 64 banks
__device__ __forceinline__ int tile_k_along(int r, int c) { return c ^ ((r >> 2) & 3); }
// position of chunk c in k-row kr of a tile with k across the rows.  16-bit: a half wave's
// transposing read takes 64 bytes (four chunks) from each of four consecutive rows, which go to different quarters of the banks; float32:
// the two half waves read rows four apart, which go to different 128-byte halves.
template <typename T> __device__ __forceinline__ int tile_k_across(int kr, int c) {
    if constexpr (sizeof(T) == 2) return c ^ ((kr & 3) << 2);
    else return c ^ (((kr >> 2) & 1) << 3);
}

typedef __attribute__((address_space(3))) char lds_char;

// 16 bytes per lane from `base` + `off` (bytes) to LDS at `dst` (the same for the whole wave, as `base`) + 16 lane.  In
// assembly because the compiler makes every LDS read behind the builtin wait for all of these loads; here wait_loads()
// counts them.  The statement has no output registers, and its wait on M0 is inside it.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t off, int dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// One operand's tile: ROWS rows (m or n) by ROW_BYTES of k.  ACROSS: k runs across the rows of memory.
template <typename T, int MODE, bool IS_B, int ROWS, int THREADS>
struct Tile {
    static constexpr int CE = Chunk<T>::n;
    static constexpr int BK = ROW_BYTES / (int)sizeof(T);
    static constexpr bool ACROSS = MODE == DW || (MODE == DX && IS_B);
    static constexpr int CHUNKS = ROWS * (ROW_BYTES / 16);
    static constexpr int PER = CHUNKS / THREADS;
    static constexpr int CPR = ACROSS ? ROWS / CE : ROW_BYTES / 16;         // chunks of a memory row
    static_assert(CHUNKS % THREADS == 0, "whole chunks per thread");

    // chunk q of the tile: (row of memory, first element in it, both inside the tile)
    static __device__ __forceinline__ void place(int q, int& r, int& e) {
        r = q / CPR;
        const int pos = q % CPR;
        e = (ACROSS ? tile_k_across<T>(r, pos) : tile_k_along(r, pos)) * CE;
    }
    // address of memory row `r` of the tile that starts at (row0, k0); FWD's B: groups of 32 rows, gate and up in turn.
    // Rows of m or n beyond the edge repeat the last one (their results are never stored).
    static __device__ __forceinline__ const T* row_ptr(const ProductArgs& a, int64_t row0, int64_t rows, int64_t k0, int r, bool second) {
        const Operand& o = IS_B ? a.B : a.A;
        if constexpr (ACROSS) {
            if (MODE == DX && second) return (const T*)o.p1 + (k0 + r) * o.ld1;
            return (const T*)o.p0 + (k0 + r) * o.ld0;
        } else if constexpr (MODE == FWD && IS_B) {
            const int64_t row = row0 / 2 + (r / 64) * 32 + (r & 31), rr = row < rows ? row : rows - 1;
            return (r & 32) ? (const T*)o.p1 + rr * o.ld1 : (const T*)o.p0 + rr * o.ld0;
        } else {
            const int64_t row = row0 + r, rr = row < rows ? row : rows - 1;
            return (const T*)o.p0 + rr * o.ld0 + (MODE == DX && second ? a.half : 0);
        }
    }
    // Where the thread's chunks of a stage come from: bytes from a base that is the same for the wave and moves on by
    // `step` bytes a stage.  FWD's B has two weights; the 16 rows of one load of a wave are all of one of them.
    static constexpr int BASES = MODE == FWD && IS_B ? PER : 1;
    struct Source {
        const char* base[BASES];
        uint32_t off[PER];
        int64_t step;
    };
    static __device__ __forceinline__ void source(const ProductArgs& a, int64_t row0, int64_t rows, Source& src) {
        const Operand& o = IS_B ? a.B : a.A;
        src.step = (ACROSS ? BK * o.ld0 : BK) * (int64_t)sizeof(T);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, e;
            place(i * THREADS + (int)threadIdx.x, r, e);
            int64_t at;
            if constexpr (ACROSS) {                // columns beyond the edge repeat the last chunk
                const int64_t col = row0 + e < rows ? row0 + e : (rows - 1) / CE * CE;
                at = r * o.ld0 + col - row0;
                src.base[0] = (const char*)((const T*)o.p0 + row0);
            } else if constexpr (MODE == FWD && IS_B) {
                const bool up = uniform(r & 32) != 0;
                const int64_t ld = up ? o.ld1 : o.ld0, row = row0 / 2 + (r / 64) * 32 + (r & 31), rr = row < rows ? row : rows - 1;
                at = (rr - row0 / 2) * ld + e;
                src.base[i] = (const char*)((const T*)(up ? o.p1 : o.p0) + row0 / 2 * ld);
            } else {
                const int64_t row = row0 + r, rr = row < rows ? row : rows - 1;
                at = (rr - row0) * o.ld0 + e;
                src.base[0] = (const char*)((const T*)o.p0 + row0 * o.ld0);
            }
            src.off[i] = (uint32_t)(at * (int64_t)sizeof(T));
        }
    }
    // to whole stage n of the first pass over k, or of the second (DX: db against the second weight)
    static __device__ __forceinline__ void seek(const ProductArgs& a, int64_t row0, int n, bool second, Source& src) {
        const Operand& o = IS_B ? a.B : a.A;
        if (MODE == DX && second) {
            if constexpr (IS_B) src.base[0] = (const char*)((const T*)o.p1 + row0);
            else src.base[0] += a.half * (int64_t)sizeof(T);
        }
#pragma unroll
        for (int i = 0; i < BASES; ++i) src.base[i] += n * src.step;
    }
    // the next whole stage, direct global -> LDS at `lds` (+ the wave's share of it)
    static __device__ __forceinline__ void load_direct(Source& src, int lds) {
#pragma unroll
        for (int i = 0; i < PER; ++i) load_to_lds(src.base[BASES == 1 ? 0 : i], src.off[i], lds + i * THREADS * 16);
#pragma unroll
        for (int i = 0; i < BASES; ++i) src.base[i] += src.step;
    }
    // ragged stage, through registers: zeros from k = K on.  (Chunks are whole: rows along k are padded with zeros to whole
    // chunks, what is behind the edge of an across row inside its last chunk is not stored.)
    static __device__ __forceinline__ void load_masked(const ProductArgs& a, int64_t row0, int64_t rows, int64_t k0, bool second, char* lds) {
        Vec<T> v[PER];
        bool in[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, e;
            place(i * THREADS + (int)threadIdx.x, r, e);
            in[i] = ACROSS ? k0 + r < a.K && row0 + e < rows : k0 + e < a.K;
            const int64_t kk = in[i] ? k0 : 0, col = !ACROSS ? (in[i] ? k0 + e : 0) : in[i] ? row0 + e : 0;
            v[i] = load_chunk(row_ptr(a, row0, rows, kk, ACROSS && !in[i] ? 0 : r, second) + col);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
#pragma unroll
            for (int e = 0; e < CE; ++e) v[i].e[e] = in[i] ? v[i].e[e] : (T)0.0f;
            *(Vec<T>*)(lds + (size_t)(i * THREADS + threadIdx.x) * 16) = v[i];
        }
    }
    // The lane's operands: byte offsets in a stage, found once, of `N` groups of 32 rows from `base` on
    template <int N> struct Lane { int off[ACROSS ? N : 2]; };
    template <int N> static __device__ __forceinline__ void place_lane(Lane<N>& l, int base, int lane, int tile) {
        if constexpr (!ACROSS) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
                l.off[ks] = tile + (base + (lane & 31)) * ROW_BYTES + tile_k_along(lane & 31, 2 * ks + (lane >> 5)) * 16;
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if constexpr (sizeof(T) == 2) {
                    const int g = lane >> 4, i = lane & 15, kr = 8 * (g >> 1) + (i >> 2);
                    const int c = (base + 32 * n) / 8 + 2 * (g & 1) + ((i >> 1) & 1);
                    l.off[n] = tile + kr * (ROWS * 2) + tile_k_across<T>(kr, c) * 16 + (i & 1) * 8;
                } else {
                    const int m = base + 32 * n + (lane & 31), kr = 4 * (lane >> 5);
                    l.off[n] = tile + kr * (ROWS * 4) + tile_k_across<T>(kr, m >> 2) * 16 + (m & 3) * 4;
                }
            }
        }
    }
    // operand of group n for k step ks (16 elements of k, float32: 8) of the stage at `lds`
    template <int N> static __device__ __forceinline__ typename Frag<T>::type frag(const char* lds, const Lane<N>& l, int n, int ks) {
        if constexpr (!ACROSS) {
            return *(const typename Frag<T>::type*)(lds + l.off[ks] + n * 32 * ROW_BYTES);
        } else if constexpr (sizeof(T) == 2) {
            short8v out;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const char* p = lds + l.off[n] + (16 * ks + 4 * half) * (ROWS * 2);
                const short4v t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
#pragma unroll
                for (int s = 0; s < 4; ++s) out[4 * half + s] = t[s];
            }
            return out;
        } else {
            floatx4 out;
#pragma unroll
            for (int s = 0; s < 4; ++s) out[s] = *(const float*)(lds + l.off[n] + (8 * ks + s) * (ROWS * 4));
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

// until at most AHEAD - 1 stages (fewer asked for: none), of LOADS loads a thread, are under way
template <int LOADS> __device__ __forceinline__ void wait_loads(int stages) {
    if (stages >= AHEAD - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 1) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
// every wave's LDS accesses so far are done, and no wave goes on before that
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(const ProductArgs args) {
    constexpr int THREADS = WM * WN * 64;
    using TA = Tile<T, MODE, false, BM, THREADS>;
    using TB = Tile<T, MODE, true, BN, THREADS>;
    constexpr int BK = TA::BK;
    constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
    constexpr int A_BYTES = BM * ROW_BYTES, BUF = A_BYTES + BN * ROW_BYTES;
    constexpr int LOADS = TA::PER + TB::PER;
    static_assert(MODE != FWD || NI % 2 == 0, "gate and up groups in pairs");
    static_assert(BK / (sizeof(T) == 2 ? 16 : 8) == 2, "two k steps a stage");
    extern __shared__ __align__(128) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    int tm, tn;
    tile_of(blockIdx.x, args.tiles_m, args.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;              // FWD: n0 counts gate and up rows
    // Stages of k: the ragged ends first (DX: of da and of db), then the whole ones, so that all but the first few go the
    // direct way.  This block's slice of them: [first, last).
    const int whole = (int)(args.K / BK), ragged = args.K % BK ? (MODE == DX ? 2 : 1) : 0, all = ragged + whole * (MODE == DX ? 2 : 1);
    const int first = blockIdx.y * args.stages, last = first + args.stages < all ? first + args.stages : all;
    floatx16 acc[MI][NI] = {};
    typename TA::Source sa;
    typename TB::Source sb;
    TA::source(args, m0, args.M, sa);
    TB::source(args, n0, args.N, sb);
    const int wave_at = uniform((int)(uint32_t)(uintptr_t)(lds_char*)lds + wave * 1024);
    // the next whole stage in line into place `at` of the ring; DX: number `whole` begins with the second pass
    int next = first > ragged ? first - ragged : 0;
    if (MODE == DX && next >= whole) {
        TA::seek(args, m0, next - whole, true, sa);
        TB::seek(args, n0, next - whole, true, sb);
    } else {
        TA::seek(args, m0, next, false, sa);
        TB::seek(args, n0, next, false, sb);
    }
    auto load_a = [&](int at) {
        if (MODE == DX && next == whole && first - ragged < whole) {
            sa.base[0] -= whole * sa.step;
            TA::seek(args, m0, 0, true, sa);
            TB::seek(args, n0, 0, true, sb);
        }
        TA::load_direct(sa, wave_at + at);
        ++next;
    };
    auto load_b = [&](int at) { TB::load_direct(sb, wave_at + at + A_BYTES); };
    typename Frag<T>::type fa[2][MI], fb[2][NI];
    typename TA::template Lane<MI> la;
    typename TB::template Lane<NI> lb;
    TA::place_lane(la, wm * (BM / WM), lane, 0);
    TB::place_lane(lb, wn * (BN / WN), lane, A_BYTES);
    auto read = [&](const char* buf, int ks) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[ks][i] = TA::frag(buf, la, i, ks);
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[ks][j] = TB::frag(buf, lb, j, ks);
    };
    auto multiply = [&](int ks, int from, int to) {
#pragma unroll
        for (int i = from; i < to; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mma(T(), fa[ks][i], fb[ks][j], acc[i][j]);
    };
    // order of a half stage's instructions: a product first (its operands are there), then the reads among the others
    auto interleave = [&](auto rows) {
        constexpr int across = sizeof(T) == 2 ? 2 : 4;
        constexpr int READS = MI * (TA::ACROSS ? across : 1) + NI * (TB::ACROSS ? across : 1);
        constexpr int PRODUCTS = decltype(rows)::value * NI * (sizeof(T) == 4 ? 4 : 1), EACH = (READS + PRODUCTS - 2) / (PRODUCTS - 1);
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
        }
    };
    for (int t = 0; t < AHEAD && first + t < last; ++t) {
        const int s = first + t;
        char* buf = lds + t * BUF;
        if (s >= ragged) {
            load_a(t * BUF);
            load_b(t * BUF);
        } else {                                    // its loads are waited for at once, and with them all earlier ones
            TA::load_masked(args, m0, args.M, (int64_t)whole * BK, s == 1, buf);
            TB::load_masked(args, n0, args.N, (int64_t)whole * BK, s == 1, buf + A_BYTES);
        }
    }
    wait_loads<LOADS>(last - first - 1);
    lds_barrier();
    read(lds, 0);
    // One stage a turn: the products of its first half, among them A's loads of the stage three ahead and the reads of its
    // second half; the barrier; the products of the second half, which cover the first reads of the next stage and B's
    // loads (all loads at once behind the barrier: the waves hold each other up, 3 % slower).  A stage is loaded into the
    // place of the one two before: what any wave read there it had used before the last barrier.  (The last turns load
    // nothing, and the very last reads a half stage that it does not use.)
    int cur = 0, fill = AHEAD * BUF;
    for (int s = first; s < last; ++s) {
        const bool more = s + AHEAD < last;
        multiply(0, 0, 1);
        if (more) load_a(fill);
        read(lds + cur, 1);
        multiply(0, 1, MI);
        interleave(std::integral_constant<int, MI - 1>{});
        cur = cur == (STAGES - 1) * BUF ? 0 : cur + BUF;
        // stage s + 1 is there when no more than the loads of s + 2 and half of those of s + 3 are under way
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 2) * LOADS + TA::PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        multiply(1, 0, 1);
        if (more) load_b(fill);
        fill = fill == (STAGES - 1) * BUF ? 0 : fill + BUF;
        read(lds + cur, 0);
        multiply(1, 1, MI);
        interleave(std::integral_constant<int, MI - 1>{});
    }
    // Results through LDS, 32 rows of the wave at a time in a corner of its own: register v of a lane is row
    // 8 (v / 4) + 4 (lane / 32) + v % 4, column lane % 32; what leaves are 16-byte chunks of whole rows.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    constexpr int COLS = NI * 32, PITCH = COLS + 4;               // floats; the pitch spreads the rows over the banks
    static_assert(WM * WN * 32 * PITCH * 4 <= STAGES * BUF, "the corners fit");
    float* corner = (float*)lds + wave * (32 * PITCH);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) corner[(8 * (v / 4) + 4 * (lane >> 5) + v % 4) * PITCH + 32 * j + (lane & 31)] = acc[i][j][v];
        const int64_t row0 = m0 + wm * (BM / WM) + 32 * i;
        if constexpr (MODE == FWD) {
            // f and p are float32: with four columns a lane one store of theirs covers whole lines, with eight (16-bit types)
            // every other 16 bytes of twice as many (T 8192, d 2048, h 8192, bf16, step: 1615 and 1880 us).  The same width
            // where they are not kept: the compiler rounds f b to float16 in one step or in two by what is around it, and y
            // must not depend on whether f and p are kept.
            constexpr int W = 4, PER_ROW = COLS / 2 / W;
            by_act(args.act, [&](auto kind) {
                constexpr int ACT = decltype(kind)::value;
#pragma unroll 2
                for (int q = lane; q < 32 * PER_ROW; q += 64) {
                    const int r = q / PER_ROW, c = q % PER_ROW * W;                   // c: column among the wave's outputs
                    const float* g = corner + r * PITCH + c / 32 * 64 + c % 32;
                    const int64_t m = row0 + r, n = n0 / 2 + wn * (COLS / 2) + c, left = m < args.M ? args.N - n : 0;
                    if (left > 0) gate_out<T, ACT, W>(args, m * args.N + n, g, g + 32, left);
                }
            });
        } else if (args.partial) {
            constexpr int PER_ROW = COLS / 4;
            for (int q = lane; q < 32 * PER_ROW; q += 64) {
                const int r = q / PER_ROW, c = q % PER_ROW * 4;
                const int64_t m = row0 + r, n = n0 + wn * COLS + c, left = m < args.M ? args.N - n : 0;
                if (left > 0) store_part(args.partial + ((int64_t)blockIdx.y * args.M + m) * args.N + n, *(const Vec<float>*)(corner + r * PITCH + c), left);
            }
        } else {
            constexpr int CE = Chunk<T>::n, PER_ROW = COLS / CE;
#pragma unroll 2
            for (int q = lane; q < 32 * PER_ROW; q += 64) {
                const int r = q / PER_ROW, c = q % PER_ROW * CE;
                const int64_t n = n0 + wn * COLS + c;
                int64_t m = row0 + r;
                T* out = (T*)args.out0;
                if (MODE == DW && m >= args.half) { m -= args.half; out = (T*)args.out1; }
                const int64_t left = m < (MODE == DW ? args.h : args.M) ? args.N - n : 0;
                if (left <= 0) continue;
                Vec<T> o;
#pragma unroll
                for (int e = 0; e < CE; ++e) o.e[e] = from_f32<T>(corner[r * PITCH + c + e]);
                store_part(out + m * args.N + n, o, left);
            }
        }
    }
}

// Sum of the k slices [slices][2][at1 or n], rounded once: elements [0, n0) to out0, [at1, at1 + n0) to out1
template <typename T>
__global__ __launch_bounds__(256) void sum_slices_kernel(const float* __restrict__ partial, int slices, int64_t n, int64_t n0, int64_t at1, T* __restrict__ out0, T* __restrict__ out1) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        if (i >= n0 && (i < at1 || i >= at1 + n0)) continue;
        float s = 0.0f;
        for (int z = 0; z < slices; ++z) s += partial[z * n + i];
        if (i < n0) out0[i] = from_f32<T>(s);
        else out1[i - at1] = from_f32<T>(s);
    }
}

// Few rows (T <= 32 MT): the weights are read once and nothing else counts.  A block owns 32 columns j (rows of both
// weights), its eight waves split d; a lane reads 64 consecutive bytes of one weight row and of one row of x, straight
// into matrix operands (the order of k inside a run is the same for both, so it needs no shuffle).  The eight partial
// sums meet in LDS.  Narrow weights leave most CUs without a block: d is then cut into slices over blocks too, whose sums
// of a and b go to partial [slices][rows][2][h] and are finished by a second launch (5 x 3337 x 80 f16: 41 -> 22 us).
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
    for (int64_t k0 = ((int64_t)blockIdx.y * WAVES + wave) * RUN; k0 < d; k0 += (int64_t)gridDim.y * WAVES * RUN) {
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
                g[c] = load_clipped(wg, k + c * CE, d);
                u[c] = load_clipped(wu, k + c * CE, d);
#pragma unroll
                for (int i = 0; i < MT; ++i) xv[i][c] = load_clipped(x[i], k + c * CE, d);
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
    by_act(args.act, [&](auto kind) {
        constexpr int ACT = decltype(kind)::value;
        const int64_t j0 = (int64_t)blockIdx.x * 32;
        for (int q = threadIdx.x; q < MT * 32 * (32 / CE); q += 512) {
            const int t = q / (32 / CE), c = q % (32 / CE) * CE;
            if (t >= args.M || j0 + c >= args.N) continue;
            // row t is register v of half wave `half` in row tile t / 32
            const int tt = t % 32, v = 4 * (tt / 8) + tt % 4, half = (tt / 4) % 2;
            float a[CE] = {}, b[CE] = {};
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int e = 0; e < CE; ++e) {
                    a[e] += part[(((w * MT + t / 32) * 2 + 0) * 16 + v) * 64 + 32 * half + c + e];
                    b[e] += part[(((w * MT + t / 32) * 2 + 1) * 16 + v) * 64 + 32 * half + c + e];
                }
            if (args.partial == nullptr) {
                gate_out<T, ACT, CE>(args, t * args.N + j0 + c, a, b, args.N - (j0 + c));
                continue;
            }
            float* out = args.partial + (((int64_t)blockIdx.y * args.M + t) * 2) * args.N + j0 + c;
#pragma unroll
            for (int e = 0; e < CE; ++e)
                if (j0 + c + e < args.N) { out[e] = a[e]; out[args.N + e] = b[e]; }
        }
    });
}
// y (f, p) from the sums of a and b over the slices of d
template <typename T>
__global__ __launch_bounds__(256) void gated_finish_kernel(const ProductArgs args, int slices) {
    constexpr int CE = Chunk<T>::n;
    const int64_t per = (args.N + CE - 1) / CE, q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= args.M * per) return;
    const int64_t t = q / per, j = q % per * CE;
    float a[CE] = {}, b[CE] = {};
    for (int z = 0; z < slices; ++z) {
        const float* in = args.partial + (((int64_t)z * args.M + t) * 2) * args.N + j;
#pragma unroll
        for (int e = 0; e < CE; ++e)
            if (j + e < args.N) { a[e] += in[e]; b[e] += in[args.N + e]; }
    }
    by_act(args.act, [&](auto kind) { gate_out<T, decltype(kind)::value, CE>(args, t * args.N + j, a, b, args.N - j); });
}

// da = gy p and, `half` columns behind it, db = gy f of every row, both padded with zeros: bandwidth (reads of f and p in float32
// and of gy, two writes of T h elements)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void gated_da_db_kernel(const float* __restrict__ f, const float* __restrict__ p, const T* __restrict__ gy, int64_t ldgy,
                                                           T* __restrict__ dab, int64_t half, int64_t rows, int64_t h) {
    constexpr int CE = Chunk<T>::n;
    const int64_t per = (h + CE - 1) / CE;
    for (int64_t t = blockIdx.y; t < rows; t += gridDim.y)
        for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < per; q += (int64_t)gridDim.x * 256) {
            const int64_t c = q * CE;
            auto load = [&](auto* row, int64_t at) { return WHOLE ? load_chunk(row + at) : load_clipped(row, at, h); };
            Vec<float> vf[CE / 4], vp[CE / 4];
#pragma unroll
            for (int k = 0; k < CE / 4; ++k) { vf[k] = load(f + t * h, c + 4 * k); vp[k] = load(p + t * h, c + 4 * k); }
            const Vec<T> vg = load(gy + t * ldgy, c);
            Vec<T> da, db;
#pragma unroll
            for (int i = 0; i < CE; ++i) {
                const float g = to_f32(vg.e[i]);
                da.e[i] = from_f32<T>(g * vp[i / 4].e[i % 4]);
                db.e[i] = from_f32<T>(g * vf[i / 4].e[i % 4]);
            }
            *(Vec<T>*)(dab + t * 2 * half + c) = da;                // zeros behind h
            *(Vec<T>*)(dab + t * 2 * half + half + c) = db;
        }
}

// -- host ------------------------------------------------------------------------------------------------------------
struct Plan { bool big; int slices, stages; };

// Tile and split of one product.  256 x 256 tiles (one block of eight waves per CU) where they fill three quarters of the
// chip, else 128 x 128 (T 4096, d 1024, forward, large : small tiles; bf16: 128 large ones 31 : 25 us, 160 30 : 33, 192 32 : 36;
// float32: 192 241 : 209, 224 240 : 252); if those are too few for that, k is cut into slices of at least sixteen stages, up to
// one block for every CU (the gradients' products only).
// Two blocks for every CU cost more in the slices' sum than they save (kernel and sum, one : two blocks a CU; T 1999,
// d 1000, h 2731, float16, dx and dW: 89 : 95 us; T 32768, d 128, h 512, float32, dW: 93 : 102 us).
template <typename T> Plan plan_of(int mode, int64_t M, int64_t N, int64_t K) {
    const int cus = marl_net::device_cus(256);
    const int64_t bk = ROW_BYTES / sizeof(T), all = (K + bk - 1) / bk * (mode == DX ? 2 : 1);
    auto tiles = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
    Plan p = {tiles(256) >= cus * 3 / 4, 1, (int)all};
    if (mode != FWD && !p.big) {
        const int64_t want = cus / tiles(128), most = all / 16;
        const int64_t slices = want < 1 ? 1 : want < most ? want : most < 1 ? 1 : most;
        p.stages = (int)((all + slices - 1) / slices);
        p.slices = (int)((all + p.stages - 1) / p.stages);
    }
    return p;
}

template <typename T, int MODE, int BM, int WM, int WN>
hipError_t launch_tiles(ProductArgs& a, int64_t n_virtual, const Plan& p, hipStream_t stream) {
    static bool attr_set[marl_net::kMaxDevices];
    auto* kernel = product_kernel<T, MODE, BM, BM, WM, WN>;
    const size_t bytes = (size_t)STAGES * 2 * BM * ROW_BYTES;
    hipError_t err = marl_net::allow_dynamic_lds((const void*)kernel, bytes, attr_set);
    if (err != hipSuccess) return err;
    a.tiles_m = (int)((a.M + BM - 1) / BM);
    a.tiles_n = (int)((n_virtual + BM - 1) / BM);
    a.stages = p.stages;
    hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n, p.slices), dim3(WM * WN * 64), bytes, stream, a);
    return hipGetLastError();
}

template <typename T, int MODE>
hipError_t launch_product(ProductArgs& a, float* partial, hipStream_t stream) {
    const int64_t n_virtual = MODE == FWD ? ((a.N + 31) / 32) * 64 : a.N;       // FWD: gate and up in groups of 32
    const Plan p = plan_of<T>(MODE, a.M, n_virtual, a.K);
    a.partial = p.slices > 1 ? partial : nullptr;
    const hipError_t err = p.big ? launch_tiles<T, MODE, 256, 2, 4>(a, n_virtual, p, stream) : launch_tiles<T, MODE, 128, 2, 2>(a, n_virtual, p, stream);
    if (err != hipSuccess || a.partial == nullptr) return err;
    const int64_t n = a.M * a.N;
    const int64_t blocks = (n + 255) / 256;
    hipLaunchKernelGGL(sum_slices_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, partial, p.slices, n,
                       MODE == DW ? a.h * a.N : n, MODE == DW ? a.half * a.N : n, (T*)a.out0, (T*)a.out1);
    return hipGetLastError();
}

// Slices of d over blocks: fewer than 64 blocks of columns, and a run for every wave of every slice.  (d 4096, one slice : up to
// 128 blocks in all; bf16, T 1: 16 blocks of columns 20 : 16 us, 32 20 : 15, 48 20 : 18, 64 20 : 19, T 64: 32 32 : 23, 64 33 : 28;
// float32, T 1: 16 50 : 17, 32 52 : 21, 48 53 : 33, 64 53 : 34.  Two slices would still gain there; from 128 blocks on there is one.)
template <typename T> int few_rows_slices(int64_t d, int64_t h) {
    const int64_t blocks = (h + 31) / 32, most = d / (64 * Chunk<T>::n);
    if (blocks >= 64 || most < 2) return 1;
    return (int)(128 / blocks < most ? 128 / blocks : most);
}

template <typename T, int MT> hipError_t launch_few_rows(ProductArgs& a, void* ws, hipStream_t stream) {
    static bool attr_set[marl_net::kMaxDevices];
    const size_t bytes = (size_t)8 * MT * 2 * 16 * 64 * sizeof(float);
    hipError_t err = marl_net::allow_dynamic_lds((const void*)gated_few_rows_kernel<T, MT>, bytes, attr_set);
    if (err != hipSuccess) return err;
    const int slices = few_rows_slices<T>(a.K, a.N);
    a.partial = slices > 1 ? (float*)ws : nullptr;
    hipLaunchKernelGGL((gated_few_rows_kernel<T, MT>), dim3((unsigned)((a.N + 31) / 32), slices), dim3(512), bytes, stream, a);
    if (slices > 1) {
        const int64_t n = a.M * ((a.N + Chunk<T>::n - 1) / Chunk<T>::n);
        hipLaunchKernelGGL(gated_finish_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a, slices);
    }
    return hipGetLastError();
}

int64_t round_256(int64_t n) { return (n + 255) / 256 * 256; }

// Rows of `n` elements as the product kernel takes them: 16-byte aligned, the last chunk whole, with zeros behind the row's end.
struct Matrix { const void* p; int64_t ld, rows; };
// (strides up to 2^21 elements: offsets inside a tile are 32-bit bytes)
constexpr int64_t MAX_LD = 1 << 21;
template <typename T> bool aligned(const Matrix& m, int64_t n) {
    return ((uintptr_t)m.p & 15) == 0 && m.ld % Chunk<T>::n == 0 && n % Chunk<T>::n == 0 && m.ld <= MAX_LD;
}
template <typename T> int64_t packed_ld(int64_t n) { return (n + Chunk<T>::n - 1) / Chunk<T>::n * Chunk<T>::n; }
template <typename T> size_t packed_bytes(const Matrix& m, int64_t n, bool always = false) {
    return aligned<T>(m, n) && !always ? 0 : (size_t)round_256(m.rows * packed_ld<T>(n) * (int64_t)sizeof(T));
}
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const T* __restrict__ src, int64_t ld, T* __restrict__ dst, int64_t rows, int64_t n, int64_t per) {
    constexpr int CE = Chunk<T>::n;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < per; q += (int64_t)gridDim.x * 256)
            *(Vec<T>*)(dst + (r * per + q) * CE) = load_clipped(src + r * ld, q * CE, n);
}
// m itself, or its copy in the workspace (which moves on)
template <typename T> Matrix pack(const Matrix& m, int64_t n, char*& ws, hipStream_t stream, bool always = false) {
    const size_t bytes = packed_bytes<T>(m, n, always);
    if (bytes == 0) return m;
    const Matrix to = {ws, packed_ld<T>(n), m.rows};
    ws += bytes;
    const int64_t per = to.ld / Chunk<T>::n;
    hipLaunchKernelGGL(pack_rows_kernel<T>, dim3((unsigned)((per + 255) / 256), (unsigned)(m.rows < 65535 ? m.rows : 65535)), dim3(256), 0, stream,
                       (const T*)m.p, m.ld, (T*)to.p, m.rows, n, per);
    return to;
}

struct Gated { int64_t rows; int32_t d, h; Matrix x, wg, wu; };
constexpr int FEW_ROWS = 64;              // up to here the forward product reads its operands as they are

template <typename T> size_t workspace(const Gated& g, bool backward) {
    const bool both = backward && (g.wg.ld != g.wu.ld || !aligned<T>(g.wg, g.d) || !aligned<T>(g.wu, g.d));
    const size_t packed = backward || g.rows > FEW_ROWS ? packed_bytes<T>(g.x, g.d) + packed_bytes<T>(g.wg, g.d, both) + packed_bytes<T>(g.wu, g.d, both) : 0;
    if (!backward) {
        const int slices = g.rows <= FEW_ROWS ? few_rows_slices<T>(g.d, g.h) : 1;
        return packed + (slices > 1 ? (size_t)slices * g.rows * 2 * g.h * sizeof(float) : 0);
    }
    const int64_t h2 = 2 * packed_ld<T>(g.h);
    const Plan px = plan_of<T>(DX, g.rows, g.d, g.h), pw = plan_of<T>(DW, h2, g.d, g.rows);
    const int64_t sx = px.slices > 1 ? px.slices * g.rows * g.d : 0, sw = pw.slices > 1 ? pw.slices * h2 * g.d : 0;
    return packed + (size_t)(round_256(g.rows * h2 * (int64_t)sizeof(T)) + (sx > sw ? sx : sw) * (int64_t)sizeof(float));
}

template <typename T> int forward(int act, Gated g, void* y, float* f, float* p, void* workspace, hipStream_t stream) {
    ProductArgs a = {};
    char* ws = (char*)workspace;
    if (g.rows > FEW_ROWS) { g.x = pack<T>(g.x, g.d, ws, stream); g.wg = pack<T>(g.wg, g.d, ws, stream); g.wu = pack<T>(g.wu, g.d, ws, stream); }
    a.A = {g.x.p, nullptr, g.x.ld, 0};
    a.B = {g.wg.p, g.wu.p, g.wg.ld, g.wu.ld};
    a.M = g.rows; a.N = g.h; a.K = g.d; a.h = g.h;
    a.out0 = y; a.save_f = f; a.save_p = p; a.act = act;
    const hipError_t err = g.rows <= 32 ? launch_few_rows<T, 1>(a, workspace, stream) : g.rows <= FEW_ROWS ? launch_few_rows<T, 2>(a, workspace, stream)
                                                                                                : launch_product<T, FWD>(a, nullptr, stream);
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

template <typename T> int backward(Gated g, const float* f, const float* p, const void* gy, int64_t ldgy, void* dx, void* dwg, void* dwu,
                                   void* workspace, hipStream_t stream) {
    char* ws = (char*)workspace;
    const int64_t half = packed_ld<T>(g.h), per = half / Chunk<T>::n;
    T* dab = (T*)ws;
    ws += round_256(g.rows * 2 * half * (int64_t)sizeof(T));
    auto* da_db = g.h % Chunk<T>::n == 0 ? gated_da_db_kernel<T, true> : gated_da_db_kernel<T, false>;
    hipLaunchKernelGGL(da_db, dim3((unsigned)((per + 255) / 256), (unsigned)(g.rows < 65535 ? g.rows : 65535)), dim3(256), 0, stream,
                       f, p, (const T*)gy, ldgy, dab, half, g.rows, (int64_t)g.h);
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && dx) {                // DX moves through both weights with one stride
        const bool both = g.wg.ld != g.wu.ld || !aligned<T>(g.wg, g.d) || !aligned<T>(g.wu, g.d);
        g.wg = pack<T>(g.wg, g.d, ws, stream, both);
        g.wu = pack<T>(g.wu, g.d, ws, stream, both);
    }
    if (err == hipSuccess && dwg) g.x = pack<T>(g.x, g.d, ws, stream);
    float* partial = (float*)ws;
    if (err == hipSuccess && dx) {
        ProductArgs a = {};
        a.A = {dab, nullptr, 2 * half, 0};
        a.B = {g.wg.p, g.wu.p, g.wg.ld, g.wu.ld};
        a.M = g.rows; a.N = g.d; a.K = g.h; a.h = g.h; a.half = half; a.out0 = dx;
        err = launch_product<T, DX>(a, partial, stream);
    }
    if (err == hipSuccess && dwg) {
        ProductArgs a = {};
        a.A = {dab, nullptr, 2 * half, 0};
        a.B = {g.x.p, nullptr, g.x.ld, 0};
        a.M = 2 * half; a.N = g.d; a.K = g.rows; a.h = g.h; a.half = half; a.out0 = dwg; a.out1 = dwu;
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
    if (rows > (1ll << 31) - 256 || d > (1 << 20) || h > (1 << 20) || ((rows + 127) / 128) * (((int64_t)h + 31) / 32) > (1ll << 30) ||
        ((rows + 127) / 128) * (((int64_t)d + 31) / 32) > (1ll << 30)) return MARL_EUNSUPPORTED;
    return MARL_OK;
}

}  // namespace

extern "C" {

int marl_gated_forward(int32_t dtype, int32_t act, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* w_gate,
                       int64_t ld_gate, const void* w_up, int64_t ld_up, void* y, float* f, float* p, void* workspace_, void* stream) {
    const int rc = check_sizes(dtype, act, rows, d, h);
    if (rc != MARL_OK) return rc;
    if (!x || !w_gate || !w_up || !y || (f == nullptr) != (p == nullptr) || ((uintptr_t)workspace_ & 15)) return MARL_EINVAL;
    if (ldx < d && rows > 1) return MARL_EINVAL;
    if ((ld_gate < d || ld_up < d) && h > 1) return MARL_EINVAL;
    const Gated g = {rows, d, h, {x, ldx, rows}, {w_gate, ld_gate, h}, {w_up, ld_up, h}};
    if (!workspace_ && MARL_BY_TYPE(dtype, workspace, g, false) > 0) return MARL_EINVAL;
    return MARL_BY_TYPE(dtype, forward, act, g, y, f, p, workspace_, (hipStream_t)stream);
}

size_t marl_gated_workspace_bytes(int32_t dtype, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* w_gate,
                                  int64_t ld_gate, const void* w_up, int64_t ld_up, int32_t backward_) {
    if (check_sizes(dtype, MARL_ACT_SILU, rows, d, h) != MARL_OK) return 0;
    const Gated g = {rows, d, h, {x, ldx, rows}, {w_gate, ld_gate, h}, {w_up, ld_up, h}};
    return MARL_BY_TYPE(dtype, workspace, g, backward_ != 0);
}

int marl_gated_backward(int32_t dtype, int64_t rows, int32_t d, int32_t h, const void* x, int64_t ldx, const void* w_gate,
                        int64_t ld_gate, const void* w_up, int64_t ld_up, const float* f, const float* p, const void* gy, int64_t ld_gy,
                        void* dx, void* dw_gate, void* dw_up, void* workspace_, void* stream) {
    const int rc = check_sizes(dtype, MARL_ACT_SILU, rows, d, h);
    if (rc != MARL_OK) return rc;
    if (!x || !w_gate || !w_up || !f || !p || !gy || !workspace_ || ((uintptr_t)workspace_ & 15) || (dw_gate == nullptr) != (dw_up == nullptr)) return MARL_EINVAL;
    if ((ldx < d || ld_gy < h) && rows > 1) return MARL_EINVAL;
    if ((ld_gate < d || ld_up < d) && h > 1) return MARL_EINVAL;
    const Gated g = {rows, d, h, {x, ldx, rows}, {w_gate, ld_gate, h}, {w_up, ld_up, h}};
    return MARL_BY_TYPE(dtype, backward, g, f, p, gy, ld_gy, dx, dw_gate, dw_up, workspace_, (hipStream_t)stream);
}

}  // extern "C"
