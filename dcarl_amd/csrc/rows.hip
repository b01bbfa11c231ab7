// Rows of a table by id, and the gradient of that table.
//   forward:  out[n] = scale * table[ids[n]], zeros where ids[n] is outside [0, S) (-1 = a visit the sampler dropped, DS:50-51)
//   gradient: grad[s] = scale * sum of dout[n] over the n with ids[n] == s, in ascending n: the ids are sorted by a stable radix sort, a row's
//             gradient is the sum over its run -- no atomics on values, run-to-run identical
// DS = Simulation_testing/Simulation_Data_Collection/Data_Sampling/data_sampling.py
#include <type_traits>
#include "seq_common.h"

namespace dcarl {

constexpr int RW_THREADS = 256;
constexpr int RW_CHUNK = 128;                  // sorted places a long run is cut into; a run of more is long
constexpr int RW_DEEP = 8;                     // rows in flight per thread of a sum
template <typename T> constexpr int RW_VEC = 16 / sizeof(T);

__device__ __forceinline__ int64_t row_id(const void* ids, int wide, int64_t n) {
    return wide ? static_cast<const int64_t*>(ids)[n] : (int64_t) static_cast<const int32_t*>(ids)[n];
}

template <typename T, int VEC> struct RowVec { T v[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ RowVec<T, VEC> row_load(const T* p) {
    RowVec<T, VEC> r;
    __builtin_memcpy(&r, p, sizeof(r));        // rows lie at any multiple of the type: an unaligned vector load
    return r;
}

// A workgroup is `lanes` threads along a row (VEC channels each) times 256 / lanes rows; blockIdx.y: 256 * VEC channels each.  The last thread
// of a row moves back to whole vectors: the same channels as its neighbour, the same values.
struct RowLane {
    int c, r, R;
    int64_t cb;
    bool live;
};
template <int VEC> __device__ __forceinline__ RowLane row_lane(int lanes, int64_t D) {
    RowLane l;
    l.R = RW_THREADS / lanes;
    l.r = (int)threadIdx.x / lanes;
    l.c = (int)threadIdx.x - l.r * lanes;
    const int64_t c0 = ((int64_t)blockIdx.y * RW_THREADS + l.c) * VEC;
    l.cb = c0 < D - VEC ? c0 : D - VEC;
    l.live = l.r < l.R && c0 < D;
    return l;
}

template <typename T, int VEC>
__global__ __launch_bounds__(RW_THREADS) void rows_gather_kernel(const T* table, int64_t ld, int64_t S, const void* ids, int wide, int64_t N,
                                                                 int64_t D, int lanes, double scale, T* out) {
    using Acc = typename SeqType<T>::Acc;
    const RowLane l = row_lane<VEC>(lanes, D);
    if (!l.live) return;
    const int64_t step = (int64_t)gridDim.x * l.R;
    for (int64_t n = (int64_t)blockIdx.x * l.R + l.r; n < N; n += step) {
        const int64_t s = row_id(ids, wide, n);
        RowVec<T, VEC> v, o;
        const bool in = s >= 0 && s < S;
        if (in) v = row_load<T, VEC>(table + s * ld + l.cb);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.v[i] = in ? narrow<T>(widen(v.v[i]) * (Acc)scale) : narrow<T>(0.0f);
        __builtin_memcpy(out + n * D + l.cb, &o, sizeof(o));
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

// adds m rows to sum, in order: row(i) is the address of the i-th; RW_DEEP of them are in flight
template <typename T, int VEC, typename Acc, typename Row> __device__ __forceinline__ void rows_add(Acc (&sum)[VEC], int64_t m, Row&& row) {
    int64_t i = 0;
    for (; i + RW_DEEP <= m; i += RW_DEEP) {
        const T* at[RW_DEEP];
        RowVec<T, VEC> v[RW_DEEP];
#pragma unroll
        for (int j = 0; j < RW_DEEP; ++j) at[j] = row(i + j);
#pragma unroll
        for (int j = 0; j < RW_DEEP; ++j) v[j] = row_load<T, VEC>(at[j]);
#pragma unroll
        for (int j = 0; j < RW_DEEP; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += widen(v[j].v[k]);
    }
    for (; i < m; ++i) {
        const RowVec<T, VEC> v = row_load<T, VEC>(row(i));
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += widen(v.v[k]);
    }
}
// the sums of the workgroup's row groups, added in their order, for the threads of group 0
template <int VEC, typename Acc> __device__ __forceinline__ void rows_join(Acc (&sum)[VEC], Acc* lds, const RowLane& l, int lanes) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VEC; ++k) lds[threadIdx.x * VEC + k] = sum[k];
    __syncthreads();
    if (l.r == 0)
        for (int r = 1; r < l.R; ++r)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += lds[(r * lanes + l.c) * VEC + k];
}

// The sums of the long runs (more than RW_CHUNK places) over one chunk of RW_CHUNK sorted places.  At most two long runs meet a chunk: the one
// of its first place (part[chunk][0]) and the one of its last (part[chunk][1]).  The workgroup's groups take a quarter, a third ... of the places each.
template <typename T, int VEC>
__global__ __launch_bounds__(RW_THREADS) void rows_chunk_kernel(const uint32_t* key, const uint32_t* begin, const uint32_t* pos, const T* dout,
                                                                int64_t ldd, int64_t N, int64_t S, int64_t D, int lanes, typename SeqType<T>::Acc* part) {
    using Acc = typename SeqType<T>::Acc;
    __shared__ Acc lds[RW_THREADS * VEC];
    const RowLane l = row_lane<VEC>(lanes, D);
    const int64_t b = (int64_t)blockIdx.x * RW_CHUNK, e = b + RW_CHUNK < N ? b + RW_CHUNK : N;
    const uint32_t first = key[b], last = key[e - 1];
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t k = slot ? last : first;
        if ((slot && last == first) || k >= S) continue;
        const int64_t rb = begin[k], re = begin[k + 1];
        if (re - rb <= RW_CHUNK) continue;
        const int64_t lo = rb > b ? rb : b, hi = re < e ? re : e;
        const int64_t each = (hi - lo + l.R - 1) / l.R, from = lo + l.r * each, to = from + each < hi ? from + each : hi;
        Acc sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0;
        if (l.live && from < to) rows_add<T, VEC>(sum, to - from, [&](int64_t i) { return dout + (int64_t)pos[from + i] * ldd + l.cb; });
        rows_join<VEC>(sum, lds, l, lanes);
        if (l.live && l.r == 0)
            for (int i = 0; i < VEC; ++i) part[((int64_t)blockIdx.x * 2 + slot) * D + l.cb + i] = sum[i];
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(RW_THREADS) void rows_sum_kernel(const uint32_t* begin, const uint32_t* pos, const T* dout, int64_t ldd, int64_t S,
                                                              int64_t D, int lanes, double scale, const typename SeqType<T>::Acc* part, T* grad) {
    using Acc = typename SeqType<T>::Acc;
    __shared__ Acc lds[RW_THREADS * VEC];
    const RowLane l = row_lane<VEC>(lanes, D);
    auto put = [&](int64_t s, const Acc(&sum)[VEC]) {
        RowVec<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.v[i] = narrow<T>(sum[i] * (Acc)scale);
        __builtin_memcpy(grad + s * D + l.cb, &o, sizeof(o));
    };
    const int64_t s0 = (int64_t)blockIdx.x * l.R;
    const int64_t s = s0 + l.r;
    Acc sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0;
    bool is_long = false;
    if (l.live && s < S) {
        const uint32_t b = begin[s], e = begin[s + 1];
        is_long = e - b > RW_CHUNK;
        if (!is_long) {
            rows_add<T, VEC>(sum, e - b, [&](int64_t i) { return dout + (int64_t)pos[b + i] * ldd + l.cb; });
            put(s, sum);
        }
    }
    if (!__syncthreads_or(is_long)) return;
    for (int r = 0; r < l.R && s0 + r < S; ++r) {          // the long ones, the whole workgroup at each: partial sums of their chunks
        const int64_t b = begin[s0 + r], e = begin[s0 + r + 1];
        if (e - b <= RW_CHUNK) continue;
        const int64_t c0 = b / RW_CHUNK, m = (e - 1) / RW_CHUNK - c0 + 1;
        const int64_t each = (m + l.R - 1) / l.R, from = l.r * each, to = from + each < m ? from + each : m;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0;
        if (l.live && from < to)
            rows_add<Acc, VEC>(sum, to - from, [&](int64_t i) { return part + ((c0 + from + i) * 2 + (from + i == 0 && b % RW_CHUNK != 0)) * D + l.cb; });
        rows_join<VEC>(sum, lds, l, lanes);
        if (l.live && l.r == 0) put(s0 + r, sum);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
struct RowsPlan {
    int nblk, passes;
    int64_t key0, key1, pos0, pos1, hist, total, begin, part, bytes;
};
static int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }
static RowsPlan rows_plan(int64_t N, int64_t S, int64_t D, int type) {
    RowsPlan p;
    p.nblk = (int)((N + RS_ITEMS - 1) / RS_ITEMS);
    int bits = 1;
    while (bits < 32 && (S >> bits)) ++bits;
    p.passes = (bits + RS_BITS - 1) / RS_BITS;
    int64_t at = 0;
    auto take = [&](int64_t words) { const int64_t here = at; at += up16(words * 4); return here; };
    p.key0 = take(N); p.key1 = take(N); p.pos0 = take(N); p.pos1 = take(N);
    p.hist = take((int64_t)RS_BINS * p.nblk); p.total = take(RS_BINS); p.begin = take(S + 1);
    p.part = take((N + RW_CHUNK - 1) / RW_CHUNK * 2 * D * (type == DCARL_F64 ? 2 : 1));
    p.bytes = at;
    return p;
}
int64_t rows_workspace_bytes(int64_t N, int64_t S, int64_t D, int type) { return rows_plan(N, S, D, type).bytes; }

// f(T{}, VEC, threads along a row, blocks along a row)
template <typename F> static void rows_with(int type, int64_t D, F&& f) {
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto V) {
            const int64_t vecs = (D + V() - 1) / V();
            f(t, V, (int)(vecs < RW_THREADS ? vecs : RW_THREADS), (unsigned)((vecs + RW_THREADS - 1) / RW_THREADS));
        };
        if (D >= RW_VEC<T>) go(std::integral_constant<int, RW_VEC<T>>{});
        else go(std::integral_constant<int, 1>{});
    });
}

void launch_rows_gather(int type, const void* table, int64_t ld, int64_t S, const void* ids, int id_bytes, int64_t N, int64_t D, double scale,
                        void* out, hipStream_t st) {
    rows_with(type, D, [&](auto t, auto V, int lanes, unsigned across) {
        using T = decltype(t);
        const int64_t need = (N + RW_THREADS / lanes - 1) / (RW_THREADS / lanes);
        hipLaunchKernelGGL((rows_gather_kernel<T, V()>), dim3((unsigned)(need < (1 << 20) ? need : 1 << 20), across), dim3(RW_THREADS), 0, st,
                           (const T*)table, ld, S, ids, id_bytes == 8, N, D, lanes, scale, (T*)out);
    });
}

void launch_rows_gradient(int type, const void* dout, int64_t ldd, const void* ids, int id_bytes, int64_t N, int64_t D, int64_t S, double scale,
                          void* ws, void* grad, hipStream_t st) {
    const RowsPlan p = rows_plan(N, S, D, type);
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
    rows_with(type, D, [&](auto t, auto V, int lanes, unsigned across) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        Acc* part = reinterpret_cast<Acc*>(w + p.part);
        const int64_t R = RW_THREADS / lanes;
        if (N > RW_CHUNK)
            hipLaunchKernelGGL((rows_chunk_kernel<T, V()>), dim3((unsigned)((N + RW_CHUNK - 1) / RW_CHUNK), across), dim3(RW_THREADS), 0, st, k_in,
                               at(p.begin), p_in, (const T*)dout, ldd, N, S, D, lanes, part);
        hipLaunchKernelGGL((rows_sum_kernel<T, V()>), dim3((unsigned)((S + R - 1) / R), across), dim3(RW_THREADS), 0, st, at(p.begin), p_in,
                           (const T*)dout, ldd, S, D, lanes, scale, part, (T*)grad);
    });
}

}  // namespace dcarl
