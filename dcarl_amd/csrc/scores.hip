// Candidate scores adjusted by what was taken already, by biases and by masks; one row of scores per observation:
//   z = s;  taken before: z = z > 0 ? z / r : z * r;  z -= f * n + p * [n > 0];  z += bias;  not allowed: z = -inf
// n counts the row's own choices (the entries of its history behind the first given[b]), "taken before" looks at the whole history.
// Bound by memory: scores, biases and mask bits once in, scores once out.  A row's history is read by every tile of the row (from the caches) and counted in LDS, so
// no counts go through memory; what it costs is the wait for it.  256 rows of 151643 f32 with biases and masks: 86 us (5.5 TB/s) without history, 105 with 1000
// entries a row on average, 129 with 8000.
#include <type_traits>
#include "seq_common.h"

namespace dcarl {

constexpr int SC_EPT = 8;                      // candidates per thread: 16 and 32 take registers that waiting workgroups need (10 and 34 % more time without history)
constexpr uint32_t SC_SEEN = 0x80000000u;
template <typename T> constexpr int SC_VEC = 16 / sizeof(T);

struct ScoreArgs {
    const void* taken;
    const int64_t* off;
    const int32_t* given;
    const float *rep, *freq, *pres, *bias;
    const uint32_t* allowed;
    float rep0, freq0, pres0;
    int64_t B, V, n_taken, ld_in, ld_out, ld_bias, ld_allowed;
    int id_wide;
};

// The history [lo, hi) of a row, counted among the tile's nv candidates from v0 on; its entries before `own` were given.  16-byte loads; each thread's
// first one is issued before the scores' (loads return in order: behind them it would wait for memory, not for the cache).
template <int THREADS, typename I> struct ScoreHistory {
    static constexpr int W = 16 / sizeof(I), DEEP = 4;
    static constexpr int64_t STEP = (int64_t)THREADS * W;
    struct Ids { I v[W]; } first;
    int64_t i;
    __device__ __forceinline__ void begin(const I* taken, int64_t lo, int64_t hi) {
        i = lo + (int64_t)threadIdx.x * W;
        if (i + W <= hi) __builtin_memcpy(&first, taken + i, 16);
    }
    __device__ __forceinline__ static void one(I id, int64_t at, int64_t own, int64_t v0, int nv, uint32_t* cnt) {
        using U = std::conditional_t<sizeof(I) == 4, uint32_t, uint64_t>;
        const U v = (U)id - (U)v0;
        if (id >= 0 && v < (U)nv) {
            if (at < own) atomicOr(&cnt[v], SC_SEEN);
            else atomicAdd(&cnt[v], 1u);
        }
    }
    __device__ __forceinline__ static void vec(const Ids& t, int64_t at, int64_t own, int64_t v0, int nv, uint32_t* cnt) {
#pragma unroll
        for (int k = 0; k < W; ++k) one(t.v[k], at + k, own, v0, nv, cnt);
    }
    __device__ __forceinline__ void count(const I* taken, int64_t hi, int64_t own, int64_t v0, int nv, uint32_t* cnt) {
        if (i + W <= hi) { vec(first, i, own, v0, nv, cnt); i += STEP; }
        for (; i + (DEEP - 1) * STEP + W <= hi; i += DEEP * STEP) {
            Ids t[DEEP];
#pragma unroll
            for (int d = 0; d < DEEP; ++d) __builtin_memcpy(&t[d], taken + i + d * STEP, 16);
#pragma unroll
            for (int d = 0; d < DEEP; ++d) vec(t[d], i + d * STEP, own, v0, nv, cnt);
        }
        for (; i < hi; i += STEP) {
            if (i + W <= hi) {
                Ids t;
                __builtin_memcpy(&t, taken + i, 16);
                vec(t, i, own, v0, nv, cnt);
            } else
                for (int64_t k = i; k < hi; ++k) one(taken[k], k, own, v0, nv, cnt);
        }
    }
};

// A workgroup takes SC_EPT * THREADS candidates of a row: their scores, biases and masks are on the way while the row's history is counted in LDS.
template <typename T, typename I, int THREADS>
__global__ __launch_bounds__(THREADS) void scores_kernel(const T* in, T* out, ScoreArgs a) {
    constexpr int VEC = SC_VEC<T>, PIECES = SC_EPT / VEC, TILE = SC_EPT * THREADS;
    struct Raw { T v[VEC]; };
    __shared__ uint4 cnt4[TILE / 4];                       // bit 31: given, the rest: times chosen
    uint32_t* cnt = reinterpret_cast<uint32_t*>(cnt4);
    const int64_t v0 = (int64_t)blockIdx.x * TILE;
    const int nv = (int)(a.V - v0 < TILE ? a.V - v0 : TILE);
    for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
        const T* src = in + b * a.ld_in + v0;
        T* dst = out + b * a.ld_out + v0;
        int64_t lo = 0, hi = 0;
        if (a.off) {
            lo = a.off[b]; hi = a.off[b + 1];
            lo = lo < 0 ? 0 : lo > a.n_taken ? a.n_taken : lo;
            hi = hi < lo ? lo : hi > a.n_taken ? a.n_taken : hi;
        }
        const I* taken = static_cast<const I*>(a.taken);
        ScoreHistory<THREADS, I> ids;
        if (lo < hi) ids.begin(taken, lo, hi);
        Raw raw[PIECES];
        float add[PIECES][VEC];
        uint32_t bits[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int i = (p * THREADS + (int)threadIdx.x) * VEC;
            bits[p] = ~0u;                                 // VEC candidates lie in one word
            if (a.allowed && i < nv) bits[p] = a.allowed[b * a.ld_allowed + ((v0 + i) >> 5)] >> ((v0 + i) & 31);
            if (a.bias) {
                const float* bias = a.bias + b * a.ld_bias + v0 + i;
                if (i + VEC <= nv) __builtin_memcpy(add[p], bias, sizeof(add[p]));
                else
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (i + k < nv) add[p][k] = bias[k];
            }
            if (i + VEC <= nv) __builtin_memcpy(&raw[p], src + i, sizeof(Raw));
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (i + k < nv) raw[p].v[k] = src[i + k];
        }
        if (lo < hi) {
            __syncthreads();                               // the previous row's counts have been read
            for (int i = threadIdx.x; i < TILE / 4; i += THREADS) cnt4[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            const int64_t own = lo + (a.given ? a.given[b] : 0);
            ids.count(taken, hi, own, v0, nv, cnt);
            __syncthreads();
        }
        const float r = a.rep ? a.rep[b] : a.rep0, f = a.freq ? a.freq[b] : a.freq0, p0 = a.pres ? a.pres[b] : a.pres0;
        // z / r as z * (1 / r): one rounding of 2^-24 more, and no division for each of the candidates; but for an r whose inverse f32 does not hold, or holds
        // with fewer bits (below 2^-126)
        const float inverse = 1.0f / r;
        const bool divides = !__builtin_isnormal(inverse);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int i = (p * THREADS + (int)threadIdx.x) * VEC;
            if (i >= nv) continue;
            float z[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) z[k] = widen(raw[p].v[k]);
            if (lo < hi) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const uint32_t c = cnt[i + k], n = c & ~SC_SEEN;
                    const float held = z[k] > 0.0f ? (divides ? z[k] / r : z[k] * inverse) : z[k] * r;
                    z[k] = c ? held : z[k];
                    z[k] = n ? z[k] - f * (float)n - p0 : z[k];
                }
            }
            if (a.bias) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[k] += add[p][k];
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) z[k] = bits[p] >> k & 1 ? z[k] : -__builtin_inff();
            Raw o;
#pragma unroll
            for (int k = 0; k < VEC; ++k) o.v[k] = narrow<T>(z[k]);
            if (i + VEC <= nv) __builtin_memcpy(dst + i, &o, sizeof(Raw));
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (i + k < nv) dst[i + k] = o.v[k];
        }
    }
}

void launch_scores(const dcarl_scores_t& s, void* out, int64_t ld_out, hipStream_t st) {
    const ScoreArgs a{s.taken, s.taken_off, s.given, s.repetition, s.frequency, s.presence, s.bias, s.allowed, s.repetition_value, s.frequency_value,
                      s.presence_value, s.B, s.V, s.n_taken, s.ld_scores, ld_out, s.ld_bias, s.ld_allowed, s.id_bytes == 8};
    with_type(s.type, [&](auto t) {
        using T = decltype(t);
        if constexpr (!__is_same(T, double)) {
            const unsigned rows = (unsigned)(s.B < 65535 ? s.B : 65535);
            auto go = [&](auto threads) {
                constexpr int tile = SC_EPT * threads();
                const dim3 grid((unsigned)((s.V + tile - 1) / tile), rows);
                if (a.id_wide) hipLaunchKernelGGL((scores_kernel<T, int64_t, threads()>), grid, dim3(threads()), 0, st, (const T*)s.scores, (T*)out, a);
                else hipLaunchKernelGGL((scores_kernel<T, int32_t, threads()>), grid, dim3(threads()), 0, st, (const T*)s.scores, (T*)out, a);
            };
            // Every tile reads the whole history of its row.  512 threads read it half as often, 256 leave more workgroups to wait side by side:
            // 256 rows of 151643 f32, histories of 1000 on average: 105 (256) and 106 us (512); of 2000: 114 and 110; of 8000: 145 and 129.
            using std::integral_constant;
            if (s.taken_off && s.n_taken / s.B >= 1536) go(integral_constant<int, 512>{});
            else go(integral_constant<int, 256>{});
        }
    });
}

}  // namespace dcarl
