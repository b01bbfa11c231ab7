// Rows of a table by id, and the gradient of that table.
//   forward:  out[n] = scale * table[ids[n]], zeros where ids[n] is outside [0, S) (-1 = a visit the sampler dropped, DS:50-51)
//   gradient: grad[s] = scale * sum of dout[n] over the n with ids[n] == s, in ascending n: the ids are sorted by a stable radix sort, a row's
//             gradient is the sum over its run -- no atomics on values, run-to-run identical
// DS = Simulation_testing/Simulation_Data_Collection/Data_Sampling/data_sampling.py
#include "seq_common.h"

namespace dcarl {

constexpr int RW_THREADS = 256;

__device__ __forceinline__ int64_t row_id(const void* ids, int wide, int64_t n) {
    return wide ? static_cast<const int64_t*>(ids)[n] : (int64_t) static_cast<const int32_t*>(ids)[n];
}

template <typename T>
__global__ __launch_bounds__(RW_THREADS) void rows_gather_kernel(const T* table, int64_t ld, int64_t S, const void* ids, int wide, int64_t N,
                                                                 int64_t D, double scale, T* out) {
    using Acc = typename SeqType<T>::Acc;
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const int64_t s = row_id(ids, wide, n);
        const bool in = s >= 0 && s < S;
        for (int64_t d = threadIdx.x; d < D; d += RW_THREADS)
            out[n * D + d] = narrow<T>(in ? widen(table[s * ld + d]) * (Acc)scale : Acc(0));
    }
}

// ---- stable radix sort of (id, n): per pass a histogram per block, an exclusive scan of each digit over the blocks, a scatter ------------
constexpr int RS_ITEMS = 4096;                 // per block: 4 wavefronts, 1024 consecutive items each, 64 at a time
constexpr int RS_BITS = 8, RS_BINS = 1 << RS_BITS;

// the sort key: the id, or S ("no row", behind every row) for ids outside the table
__device__ __forceinline__ uint32_t row_key(const void* ids, int wide, const uint32_t* key, int64_t S, int64_t n) {
    if (key) return key[n];
    const int64_t s = row_id(ids, wide, n);
    return (uint32_t)(s >= 0 && s < S ? s : S);
}

__global__ __launch_bounds__(256) void rows_hist_kernel(const void* ids, int wide, const uint32_t* key, int64_t S, int64_t N, int shift,
                                                        uint32_t* hist, int nblk) {
    __shared__ uint32_t h[RS_BINS];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b = (int64_t)blockIdx.x * RS_ITEMS;
    for (int i = threadIdx.x; i < RS_ITEMS && b + i < N; i += 256)
        atomicAdd(&h[(row_key(ids, wide, key, S, b + i) >> shift) & (RS_BINS - 1)], 1u);
    __syncthreads();
    hist[(int64_t)threadIdx.x * nblk + blockIdx.x] = h[threadIdx.x];
}

// block d: exclusive scan of digit d's counts over the blocks, in place; its total
__global__ __launch_bounds__(256) void rows_scan_kernel(uint32_t* hist, int nblk, uint32_t* total) {
    __shared__ uint32_t sm[256];
    uint32_t* row = hist + (int64_t)blockIdx.x * nblk;
    uint32_t carry = 0;
    for (int base = 0; base < nblk; base += 256) {
        const int i = base + threadIdx.x;
        const uint32_t v = i < nblk ? row[i] : 0;
        sm[threadIdx.x] = v;
        __syncthreads();
        for (int o = 1; o < 256; o <<= 1) {
            const uint32_t add = (int)threadIdx.x >= o ? sm[threadIdx.x - o] : 0;
            __syncthreads();
            sm[threadIdx.x] += add;
            __syncthreads();
        }
        if (i < nblk) row[i] = carry + sm[threadIdx.x] - v;
        carry += sm[255];
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void rows_scatter_kernel(const void* ids, int wide, const uint32_t* key, const uint32_t* pos, int64_t S,
                                                           int64_t N, int shift, const uint32_t* hist, const uint32_t* total, int nblk,
                                                           uint32_t* key_out, uint32_t* pos_out) {
    __shared__ uint32_t cnt[4][RS_BINS];       // first the wavefronts' counts, then where each one's items of a digit go
    __shared__ uint32_t sm[RS_BINS];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
    sm[tid] = total[tid];
    __syncthreads();
    for (int o = 1; o < RS_BINS; o <<= 1) {    // inclusive scan of the digits' totals
        const uint32_t add = tid >= o ? sm[tid - o] : 0;
        __syncthreads();
        sm[tid] += add;
        __syncthreads();
    }
    const int64_t b = (int64_t)blockIdx.x * RS_ITEMS + wv * (RS_ITEMS / 4);
    for (int r = 0; r < RS_ITEMS / 256; ++r) {
        const int64_t n = b + r * 64 + lane;
        if (n < N) atomicAdd(&cnt[wv][(row_key(ids, wide, key, S, n) >> shift) & (RS_BINS - 1)], 1u);
    }
    __syncthreads();
    {
        uint32_t at = (tid ? sm[tid - 1] : 0) + hist[(int64_t)tid * nblk + blockIdx.x];
#pragma unroll
        for (int w = 0; w < 4; ++w) { const uint32_t c = cnt[w][tid]; cnt[w][tid] = at; at += c; }
    }
    __syncthreads();
    for (int r = 0; r < RS_ITEMS / 256; ++r) {
        const int64_t n = b + r * 64 + lane;
        const bool live = n < N;
        const uint32_t k = live ? row_key(ids, wide, key, S, n) : 0xffffffffu;
        const uint32_t dig = (k >> shift) & (RS_BINS - 1);
        unsigned long long same = __ballot(live);
#pragma unroll
        for (int j = 0; j < RS_BITS; ++j) {
            const unsigned long long bit = __ballot((dig >> j) & 1);
            same &= (dig >> j) & 1 ? bit : ~bit;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        uint32_t at = 0;
        if (live) at = cnt[wv][dig];
        __builtin_amdgcn_wave_barrier();       // every lane has read its digit's place before the first lane of a group moves it on
        if (live && rank == 0) cnt[wv][dig] = at + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (live) {
            key_out[at + rank] = k;
            pos_out[at + rank] = pos ? pos[n] : (uint32_t)n;
        }
    }
}

// begin[s] = first place of the sorted keys that is not below s, for s = 0 .. S
__global__ __launch_bounds__(256) void rows_begin_kernel(const uint32_t* key, int64_t N, int64_t S, uint32_t* begin) {
    const int64_t s = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (s > S) return;
    int64_t lo = 0, hi = N;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (key[mid] < (uint32_t)s) lo = mid + 1; else hi = mid;
    }
    begin[s] = (uint32_t)lo;
}

template <typename T>
__global__ __launch_bounds__(RW_THREADS) void rows_sum_kernel(const uint32_t* begin, const uint32_t* pos, const T* dout, int64_t ldd, int64_t S,
                                                              int64_t D, double scale, T* grad) {
    using Acc = typename SeqType<T>::Acc;
    for (int64_t s = blockIdx.x; s < S; s += gridDim.x) {
        const uint32_t b = begin[s], e = begin[s + 1];
        for (int64_t d = threadIdx.x; d < D; d += RW_THREADS) {
            Acc sum = 0;
            for (uint32_t i = b; i < e; ++i) sum += widen(dout[(int64_t)pos[i] * ldd + d]);
            grad[s * D + d] = narrow<T>(sum * (Acc)scale);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
struct RowsPlan {
    int nblk, passes;
    int64_t key0, key1, pos0, pos1, hist, total, begin, bytes;
};
static int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }
static RowsPlan rows_plan(int64_t N, int64_t S, int64_t) {
    RowsPlan p;
    p.nblk = (int)((N + RS_ITEMS - 1) / RS_ITEMS);
    int bits = 1;
    while (bits < 32 && (S >> bits)) ++bits;
    p.passes = (bits + RS_BITS - 1) / RS_BITS;
    int64_t at = 0;
    auto take = [&](int64_t words) { const int64_t here = at; at += up16(words * 4); return here; };
    p.key0 = take(N); p.key1 = take(N); p.pos0 = take(N); p.pos1 = take(N);
    p.hist = take((int64_t)RS_BINS * p.nblk); p.total = take(RS_BINS); p.begin = take(S + 1);
    p.bytes = at;
    return p;
}
int64_t rows_workspace_bytes(int64_t N, int64_t S, int64_t D) { return rows_plan(N, S, D).bytes; }

void launch_rows_gather(int type, const void* table, int64_t ld, int64_t S, const void* ids, int id_bytes, int64_t N, int64_t D, double scale,
                        void* out, hipStream_t st) {
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((rows_gather_kernel<T>), dim3((unsigned)(N < 65536 ? N : 65536)), dim3(RW_THREADS), 0, st, (const T*)table, ld, S, ids,
                           id_bytes == 8, N, D, scale, (T*)out);
    });
}

void launch_rows_gradient(int type, const void* dout, int64_t ldd, const void* ids, int id_bytes, int64_t N, int64_t D, int64_t S, double scale,
                          void* ws, void* grad, hipStream_t st) {
    const RowsPlan p = rows_plan(N, S, D);
    char* w = static_cast<char*>(ws);
    auto at = [&](int64_t off) { return reinterpret_cast<uint32_t*>(w + off); };
    uint32_t *k_in = nullptr, *p_in = nullptr, *k_out = at(p.key0), *p_out = at(p.pos0);
    for (int i = 0; i < p.passes && N > 0; ++i) {
        hipLaunchKernelGGL(rows_hist_kernel, dim3(p.nblk), dim3(256), 0, st, ids, id_bytes == 8, k_in, S, N, i * RS_BITS, at(p.hist), p.nblk);
        hipLaunchKernelGGL(rows_scan_kernel, dim3(RS_BINS), dim3(256), 0, st, at(p.hist), p.nblk, at(p.total));
        hipLaunchKernelGGL(rows_scatter_kernel, dim3(p.nblk), dim3(256), 0, st, ids, id_bytes == 8, k_in, p_in, S, N, i * RS_BITS, at(p.hist),
                           at(p.total), p.nblk, k_out, p_out);
        k_in = k_out; p_in = p_out;
        k_out = at(i % 2 ? p.key0 : p.key1); p_out = at(i % 2 ? p.pos0 : p.pos1);
    }
    hipLaunchKernelGGL(rows_begin_kernel, dim3((unsigned)((S + 256) / 256)), dim3(256), 0, st, k_in, N, S, at(p.begin));
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((rows_sum_kernel<T>), dim3((unsigned)(S < 65536 ? S : 65536)), dim3(RW_THREADS), 0, st, at(p.begin), p_in, (const T*)dout,
                           ldd, S, D, scale, (T*)grad);
    });
}

}  // namespace dcarl
