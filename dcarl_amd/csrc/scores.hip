// Candidate scores adjusted by what was taken already, by biases and by masks; one row of scores per observation:
//   z = s;  taken before: z = z > 0 ? z / r : z * r;  z -= f * n + p * [n > 0];  z += bias;  not allowed: z = -inf
// n counts the row's own choices (the entries of its history behind the first given[b]), "taken before" looks at the whole history.
#include "seq_common.h"

namespace dcarl {

constexpr int SC_THREADS = 256, SC_TILE = 4096;
constexpr uint32_t SC_SEEN = 0x80000000u;

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

template <typename T>
__global__ __launch_bounds__(SC_THREADS) void scores_kernel(const T* in, T* out, ScoreArgs a) {
    __shared__ uint32_t cnt[SC_TILE];          // bit 31: given, the rest: times chosen
    const int64_t v0 = (int64_t)blockIdx.x * SC_TILE;
    const int nv = (int)(a.V - v0 < SC_TILE ? a.V - v0 : SC_TILE);
    for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y) {
    __syncthreads();                           // the previous row's counts have been read
    int64_t lo = 0, hi = 0;
    if (a.off) {
        lo = a.off[b]; hi = a.off[b + 1];
        lo = lo < 0 ? 0 : lo > a.n_taken ? a.n_taken : lo;
        hi = hi < lo ? lo : hi > a.n_taken ? a.n_taken : hi;
    }
    if (lo < hi) {
        for (int i = threadIdx.x; i < nv; i += SC_THREADS) cnt[i] = 0;
        __syncthreads();
        const int64_t own = lo + (a.given ? a.given[b] : 0);
        for (int64_t i = lo + threadIdx.x; i < hi; i += SC_THREADS) {
            const int64_t v = (a.id_wide ? static_cast<const int64_t*>(a.taken)[i] : (int64_t) static_cast<const int32_t*>(a.taken)[i]) - v0;
            if (v >= 0 && v < nv) {
                if (i < own) atomicOr(&cnt[v], SC_SEEN);
                else atomicAdd(&cnt[v], 1u);
            }
        }
        __syncthreads();
    }
    const float r = a.rep ? a.rep[b] : a.rep0, f = a.freq ? a.freq[b] : a.freq0, p = a.pres ? a.pres[b] : a.pres0;
    for (int i = threadIdx.x; i < nv; i += SC_THREADS) {
        const int64_t v = v0 + i;
        float z = widen(in[b * a.ld_in + v]);
        if (lo < hi) {
            const uint32_t c = cnt[i], n = c & ~SC_SEEN;
            if (c) z = z > 0.0f ? z / r : z * r;
            if (n) z = z - f * (float)n - p;
        }
        if (a.bias) z += a.bias[b * a.ld_bias + v];
        if (a.allowed && !(a.allowed[b * a.ld_allowed + (v >> 5)] >> (v & 31) & 1)) z = -__builtin_inff();
        out[b * a.ld_out + v] = narrow<T>(z);
    }
    }
}

void launch_scores(const dcarl_scores_t& s, void* out, int64_t ld_out, hipStream_t st) {
    const ScoreArgs a{s.taken, s.taken_off, s.given, s.repetition, s.frequency, s.presence, s.bias, s.allowed, s.repetition_value, s.frequency_value,
                      s.presence_value, s.B, s.V, s.n_taken, s.ld_scores, ld_out, s.ld_bias, s.ld_allowed, s.id_bytes == 8};
    with_type(s.type, [&](auto t) {
        using T = decltype(t);
        if constexpr (!__is_same(T, double))
            hipLaunchKernelGGL((scores_kernel<T>), dim3((unsigned)((s.V + SC_TILE - 1) / SC_TILE), (unsigned)(s.B < 65535 ? s.B : 65535)), dim3(SC_THREADS), 0, st,
                               (const T*)s.scores, (T*)out, a);
    });
}

}  // namespace dcarl
