// Candidate scores adjusted by what was taken already, by biases and by masks; one row of scores per observation:
//   z = s;  taken before: z = z > 0 ? z / r : z * r;  z -= f * n + p * [n > 0];  z += bias;  not allowed: z = -inf
// n counts the row's own choices (the entries of its history behind the first given[b]), "taken before" looks at the whole history.
#include <type_traits>
#include "seq_common.h"

namespace dcarl {

constexpr int SC_THREADS = 256;
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

template <typename I> struct SixteenBytes { I v[16 / sizeof(I)]; };

// counts the history [lo, hi) of a row among the tile's nv candidates from v0 on; its entries before `own` were given
template <typename I>
__device__ __forceinline__ void scores_count(const I* taken, int64_t lo, int64_t hi, int64_t own, int64_t v0, int nv, uint32_t* cnt) {
    constexpr int W = 16 / sizeof(I), DEEP = 4;            // 16-byte loads, four in flight: 4096 entries of 32 bits a trip
    auto one = [&](I id, int64_t i) {
        const uint64_t v = (uint64_t)((int64_t)id - v0);
        if (v < (uint64_t)nv) {
            if (i < own) atomicOr(&cnt[v], SC_SEEN);
            else atomicAdd(&cnt[v], 1u);
        }
    };
    int64_t i = lo + threadIdx.x * W;
    constexpr int64_t STEP = (int64_t)SC_THREADS * W;
    for (; i + (DEEP - 1) * STEP + W <= hi; i += DEEP * STEP) {
        SixteenBytes<I> t[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) __builtin_memcpy(&t[d], taken + i + d * STEP, 16);
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int k = 0; k < W; ++k) one(t[d].v[k], i + d * STEP + k);
    }
    for (; i < hi; i += STEP) {
        if (i + W <= hi) {
            SixteenBytes<I> t;
            __builtin_memcpy(&t, taken + i, 16);
#pragma unroll
            for (int k = 0; k < W; ++k) one(t.v[k], i + k);
        } else
            for (int k = 0; i + k < hi; ++k) one(taken[i + k], i + k);
    }
}

// A workgroup takes EPT * 256 candidates of a row: their scores are on the way while the row's history is counted in LDS.
template <typename T, int EPT>
__global__ __launch_bounds__(SC_THREADS) void scores_kernel(const T* in, T* out, ScoreArgs a) {
    constexpr int VEC = SC_VEC<T>, PIECES = EPT / VEC, TILE = EPT * SC_THREADS;
    struct Raw { T v[VEC]; };
    __shared__ uint4 cnt4[TILE / 4];                       // bit 31: given, the rest: times chosen
    uint32_t* cnt = reinterpret_cast<uint32_t*>(cnt4);
    const int64_t v0 = (int64_t)blockIdx.x * TILE;
    const int nv = (int)(a.V - v0 < TILE ? a.V - v0 : TILE);
    for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
        const T* src = in + b * a.ld_in + v0;
        T* dst = out + b * a.ld_out + v0;
        Raw raw[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int i = (p * SC_THREADS + (int)threadIdx.x) * VEC;
            if (i + VEC <= nv) __builtin_memcpy(&raw[p], src + i, sizeof(Raw));
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (i + k < nv) raw[p].v[k] = src[i + k];
        }
        int64_t lo = 0, hi = 0;
        if (a.off) {
            lo = a.off[b]; hi = a.off[b + 1];
            lo = lo < 0 ? 0 : lo > a.n_taken ? a.n_taken : lo;
            hi = hi < lo ? lo : hi > a.n_taken ? a.n_taken : hi;
        }
        if (lo < hi) {
            __syncthreads();                               // the previous row's counts have been read
            for (int i = threadIdx.x; i < TILE / 4; i += SC_THREADS) cnt4[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            const int64_t own = lo + (a.given ? a.given[b] : 0);
            if (a.id_wide) scores_count(static_cast<const int64_t*>(a.taken), lo, hi, own, v0, nv, cnt);
            else scores_count(static_cast<const int32_t*>(a.taken), lo, hi, own, v0, nv, cnt);
            __syncthreads();
        }
        const float r = a.rep ? a.rep[b] : a.rep0, f = a.freq ? a.freq[b] : a.freq0, p0 = a.pres ? a.pres[b] : a.pres0;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int i = (p * SC_THREADS + (int)threadIdx.x) * VEC;
            if (i >= nv) continue;
            float z[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) z[k] = widen(raw[p].v[k]);
            if (lo < hi) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const uint32_t c = cnt[i + k], n = c & ~SC_SEEN;
                    if (c) z[k] = z[k] > 0.0f ? z[k] / r : z[k] * r;
                    if (n) z[k] = z[k] - f * (float)n - p0;
                }
            }
            if (a.bias) {
                const float* bias = a.bias + b * a.ld_bias + v0 + i;
                float add[VEC];
                if (i + VEC <= nv) __builtin_memcpy(add, bias, sizeof(add));
                else
#pragma unroll
                    for (int k = 0; k < VEC; ++k) add[k] = i + k < nv ? bias[k] : 0.0f;
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[k] += add[k];
            }
            if (a.allowed) {                               // VEC candidates lie in one word
                const uint32_t bits = a.allowed[b * a.ld_allowed + ((v0 + i) >> 5)] >> ((v0 + i) & 31);
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[k] = bits >> k & 1 ? z[k] : -__builtin_inff();
            }
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
            // short tiles while they are what fills the GPU, long ones (a quarter of the readings of each history) where there are enough of those
            const unsigned rows = (unsigned)(s.B < 65535 ? s.B : 65535);
            auto go = [&](auto ept) {
                constexpr int tile = ept() * SC_THREADS;
                hipLaunchKernelGGL((scores_kernel<T, ept()>), dim3((unsigned)((s.V + tile - 1) / tile), rows), dim3(SC_THREADS), 0, st,
                                   (const T*)s.scores, (T*)out, a);
            };
            if (s.B * ((s.V + 8191) / 8192) >= 1024) go(std::integral_constant<int, 32>{});
            else go(std::integral_constant<int, 8>{});
        }
    });
}

}  // namespace dcarl
