// Dropout whose mask is a function of (seed, row key, column) and is never stored:
//     y[r][j] = x[r][j] * s  if  draw(seed, key[r], j) >= threshold, else 0;   threshold = round(p 2^16), s = 2^16 / (2^16 - threshold).
// The draw is 16 bits of Philox4x32-10: counter (j / 8, STREAM_DROPOUT, key low, key high), key = seed, one call for eight
// columns.  The gradient is the same function of gy, so a backward pass, a replayed rollout or a shuffled minibatch that
// names its rows by the same keys meets the same mask.  A dropped element is 0 whatever it held.
// Bandwidth bound (one read, one write) as long as the ~100 integer instructions of a call, a quarter of them 32-bit
// multiplies, are shared by eight elements; 32-bit draws would take twice the calls.
// Measured: 65536 x 512 float32 49 us (5.5 TB/s); 4099 x 1537 bf16 8.1 us (3.1 TB/s), 6.9 us a call without the profiler.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "marl_env.h"
#include "marl_net.h"
#include "marl_rng.h"
#include "marl_types.h"

extern "C" __attribute__((visibility("hidden"))) void marl_note_hip_error(int err);     // marl_env.hip

namespace {

using namespace marl_types;
constexpr int GROUP = 8;                 // columns of one Philox call

// One group of eight columns per thread and turn.  magic = floor(2^32 / groups): q = umulhi(i, magic) is i / groups or
// one less, which the remainder shows.  WHOLE: rows of whole groups; the loads then do not branch and are under way while the
// generator runs.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void keyed_dropout_kernel(const T* __restrict__ x, int64_t ldx, T* __restrict__ y, const int64_t* __restrict__ keys,
                                                             int64_t first_row, uint32_t total, uint32_t groups, uint32_t magic, int32_t d,
                                                             uint32_t threshold, float scale, uint32_t seed_lo, uint32_t seed_hi) {
    constexpr int CE = Chunk<T>::n, CHUNKS = GROUP / CE;
    for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
        uint32_t q = __umulhi(i, magic), g = i - q * groups;
        if (g >= groups) { ++q; g -= groups; }
        const int64_t r = first_row + q;
        const int c = (int)g * GROUP;
        const T* px = x + r * ldx + c;
        T* py = y + r * d + c;
        Vec<T> v[CHUNKS];
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) v[k] = WHOLE ? load_chunk(px + k * CE) : load_part(px + k * CE, (int64_t)d - c - k * CE);
        const uint64_t key = keys ? (uint64_t)keys[r] : (uint64_t)r;
        uint32_t w[4];
        marl_rng::philox4x32(g, marl_rng::STREAM_DROPOUT, (uint32_t)key, (uint32_t)(key >> 32), seed_lo, seed_hi, w);
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
#pragma unroll
            for (int e = 0; e < CE; ++e) {
                const int col = k * CE + e;
                const uint32_t u = (col & 1) ? w[col / 2] >> 16 : w[col / 2] & 0xFFFFu;
                v[k].e[e] = u >= threshold ? from_f32<T>(to_f32(v[k].e[e]) * scale) : (T)0.0f;
            }
            if (WHOLE) store_chunk(py + k * CE, v[k]);
            else store_part(py + k * CE, v[k], (int64_t)d - c - k * CE);
        }
    }
}

template <typename T>
int run(int64_t rows, int32_t d, const void* x, int64_t ldx, void* y, const int64_t* keys, uint32_t threshold, uint64_t seed, hipStream_t stream) {
    const uint32_t groups = (uint32_t)((d + GROUP - 1) / GROUP);
    const uint32_t magic = groups == 1 ? 0xFFFFFFFFu : (uint32_t)((1ull << 32) / groups);
    const float scale = threshold < 65536 ? 65536.0f / (float)(65536 - threshold) : 0.0f;
    const int64_t per_launch = (1 << 30) / groups;                       // 32-bit group numbers
    for (int64_t first = 0; first < rows; first += per_launch) {
        const int64_t n = rows - first < per_launch ? rows - first : per_launch;
        const uint32_t total = (uint32_t)n * groups;
        const uint32_t blocks = (total + 255) / 256;
        auto* kernel = d % GROUP == 0 ? keyed_dropout_kernel<T, true> : keyed_dropout_kernel<T, false>;
        hipLaunchKernelGGL(kernel, dim3(blocks < 16384 ? blocks : 16384), dim3(256), 0, stream, (const T*)x, ldx, (T*)y, keys,
                           first, total, groups, magic, d, threshold, scale, (uint32_t)seed, (uint32_t)(seed >> 32));
    }
    const hipError_t err = hipGetLastError();
    if (err == hipSuccess) return MARL_OK;
    marl_note_hip_error((int)err);
    return MARL_EHIP;
}

}  // namespace

extern "C" int marl_keyed_dropout(int32_t dtype, int64_t rows, int32_t d, const void* x, int64_t ldx, void* y, const int64_t* keys, double p,
                                  uint64_t seed, void* stream) {
    if (rows < 1 || d < 1 || !x || !y || dtype < MARL_F32 || dtype > MARL_F16 || !(p >= 0.0 && p <= 1.0) || (ldx < d && rows > 1)) return MARL_EINVAL;
    if (rows > (1ll << 40) || d > (1 << 30)) return MARL_EUNSUPPORTED;
    const uint32_t threshold = (uint32_t)(p * 65536.0 + 0.5);
    return MARL_BY_TYPE(dtype, run, rows, d, x, ldx, y, keys, threshold, seed, (hipStream_t)stream);
}
