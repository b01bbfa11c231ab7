// Rows of a table by id, and the gradient of that table.
//   forward:  out[n] = scale * table[ids[n]], zeros where ids[n] is outside [0, S) (-1 = a visit the sampler dropped, DS:50-51)
//   gradient: grad[s] = scale * sum of dout[n] over the n with ids[n] == s, in ascending n: the ids are sorted by a stable radix sort, a row's
//             gradient is the sum over its run -- no atomics on values, run-to-run identical
//             (sums of f32 in f64 would take 103 us where the skewed case below takes 97, for an error of 3e-8 of the gradient's norm in place of 1.3e-7: a caller
//             who wants that hands over dout in f64)
// DS = Simulation_testing/Simulation_Data_Collection/Data_Sampling/data_sampling.py
// Bound by memory: rows in 16-byte pieces, each once; a thread sums a row's channels over its run in f32.  Runs are as uneven as the visits, so those of more than
// RW_CHUNK places are summed in chunks by workgroups of their own, then joined.  16384 ids of 50000 rows of 1024 bf16: gather 13 us (5.1 TB/s), sort 17, where the
// runs begin 5, chunks 7, sums and zeros 21 (6.4 TB/s); 131071 f32 rows of 257, six tenths of one id: 32, 24, 6, 23, 15.
#include <type_traits>
#include "seq_common.h"

namespace dcarl {

constexpr int RW_THREADS = 256;
constexpr int RW_CHUNK = 64;                   // sorted places a long run is cut into; a run of more is long
constexpr int RW_DEEP = 8;                     // rows in flight per thread of a sum
constexpr int RW_ROWS = 4;                     // rows per thread: in flight in the gather, one after the other in the sums
constexpr int RW_SUPER = 32;                   // chunks whose partial sums are joined first where a run has more
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

// a result that nothing here reads again: past the caches, at any alignment of the type (sums of the skewed ids above 21.5 -> 14.8 us)
typedef unsigned row_u4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, int VEC> __device__ __forceinline__ void row_store(T* p, const RowVec<T, VEC>& r) {
    if constexpr (sizeof(r) == 16) __builtin_nontemporal_store(__builtin_bit_cast(row_u4, r), reinterpret_cast<row_u4*>(p));
    else __builtin_memcpy(p, &r, sizeof(r));
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
    // four consecutive groups of rows at a time, their ids and then their rows in flight together
    const int64_t step = (int64_t)gridDim.x * l.R * RW_ROWS;
    for (int64_t n0 = (int64_t)blockIdx.x * l.R * RW_ROWS + l.r; n0 < N; n0 += step) {
        int64_t s[RW_ROWS];
        RowVec<T, VEC> v[RW_ROWS];
#pragma unroll
        for (int j = 0; j < RW_ROWS; ++j) {
            const int64_t n = n0 + j * l.R;
            s[j] = n < N ? row_id(ids, wide, n) : -1;
        }
#pragma unroll
        for (int j = 0; j < RW_ROWS; ++j)
            if (s[j] >= 0 && s[j] < S) v[j] = row_load<T, VEC>(table + s[j] * ld + l.cb);
#pragma unroll
        for (int j = 0; j < RW_ROWS; ++j) {
            const int64_t n = n0 + j * l.R;
            const bool in = s[j] >= 0 && s[j] < S;
            RowVec<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.v[i] = in ? narrow<T>(widen(v[j].v[i]) * (Acc)scale) : narrow<T>(0.0f);
            if (n < N) row_store(out + n * D + l.cb, o);
        }
    }
}

// ---- stable radix sort of (id, n): per pass a histogram per block, places by an exclusive scan over digits and blocks, a scatter -----------
// 1024 items per block: a scatter of 16384 ids takes 5.4 us with 16 blocks, it took 17 with 4 blocks of 4096.
constexpr int RS_ROUNDS = 4, RS_ITEMS = 256 * RS_ROUNDS;   // per block: 4 wavefronts of consecutive items, 64 at a time
constexpr int RS_BITS = 8, RS_BINS = 1 << RS_BITS;
constexpr int RS_DIRECT = 64;                  // up to so many blocks each scatter block adds the others' counts itself: a launch less

// the sort key: the id, or S ("no row", behind every row) for ids outside the table
__device__ __forceinline__ uint32_t row_key(const void* ids, int wide, const uint32_t* key, int64_t S, int64_t n) {
    if (key) return key[n];
    const int64_t s = row_id(ids, wide, n);
    return (uint32_t)(s >= 0 && s < S ? s : S);
}

// inclusive scan of 256 values over a workgroup of 256
__device__ __forceinline__ uint32_t scan256(uint32_t v, uint32_t (&tot)[4]) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 63) tot[wv] = v;
    __syncthreads();
    for (int w = 0; w < wv; ++w) v += tot[w];
    return v;
}

// LDS accesses of a wavefront's lanes stay on their side of this (the hardware keeps their order; it holds the compiler to it)
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where this lane's item goes: its digit's next place (place[digit], this wavefront's own) and its rank among the wavefront's items of that digit.
__device__ __forceinline__ uint32_t digit_place(uint32_t dig, bool live, int lane, uint32_t* place) {
    unsigned long long same = __ballot(live);
#pragma unroll
    for (int j = 0; j < RS_BITS; ++j) {
        const unsigned long long bit = __ballot((dig >> j) & 1);
        same &= (dig >> j) & 1 ? bit : ~bit;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    uint32_t to = 0;
    if (live) to = place[dig];
    wave_order();                              // every lane has read its digit's place before the first lane of a group moves it on
    if (live && rank == 0) place[dig] = to + (uint32_t)__popcll(same);
    wave_order();
    return to + rank;
}

// hist[block][digit]
__global__ __launch_bounds__(256) void rows_hist_kernel(const void* ids, int wide, const uint32_t* key, int64_t S, int64_t N, int shift, uint32_t* hist) {
    __shared__ uint32_t h[RS_BINS];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b = (int64_t)blockIdx.x * RS_ITEMS + threadIdx.x;
    uint32_t k[RS_ROUNDS];
#pragma unroll
    for (int i = 0; i < RS_ROUNDS; ++i)
        if (b + i * 256 < N) k[i] = row_key(ids, wide, key, S, b + i * 256);
#pragma unroll
    for (int i = 0; i < RS_ROUNDS; ++i)
        if (b + i * 256 < N) atomicAdd(&h[(k[i] >> shift) & (RS_BINS - 1)], 1u);
    __syncthreads();
    hist[(int64_t)blockIdx.x * RS_BINS + threadIdx.x] = h[threadIdx.x];
}

// block d: exclusive scan of digit d's counts over the blocks, in place; its total
__global__ __launch_bounds__(256) void rows_scan_kernel(uint32_t* hist, int nblk, uint32_t* total) {
    __shared__ uint32_t tot[4];
    uint32_t* col = hist + blockIdx.x;
    uint32_t carry = 0;
    for (int base = 0; base < nblk; base += 256) {
        const int i = base + threadIdx.x;
        const uint32_t v = i < nblk ? col[(int64_t)i * RS_BINS] : 0, in = scan256(v, tot);
        if (i < nblk) col[(int64_t)i * RS_BINS] = carry + in - v;
        __syncthreads();
        carry += tot[0] + tot[1] + tot[2] + tot[3];
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// total == NULL: hist holds the blocks' own counts, nblk <= RS_DIRECT
__global__ __launch_bounds__(256) void rows_scatter_kernel(const void* ids, int wide, const uint32_t* key, const uint32_t* pos, int64_t S,
                                                           int64_t N, int shift, const uint32_t* hist, const uint32_t* total, int nblk,
                                                           uint32_t* key_out, uint32_t* pos_out) {
    __shared__ uint32_t cnt[4][RS_BINS];       // first the wavefronts' counts, then where each one's items of a digit go
    __shared__ uint32_t tot[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t b = (int64_t)blockIdx.x * RS_ITEMS + wv * (64 * RS_ROUNDS) + lane;
    uint32_t k[RS_ROUNDS], ps[RS_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const int64_t n = b + r * 64;
        k[r] = n < N ? row_key(ids, wide, key, S, n) : 0xffffffffu;
        ps[r] = n < N && pos ? pos[n] : (uint32_t)n;
    }
    uint32_t all = 0, before = 0;              // of digit `tid`: items everywhere, items in earlier blocks
    if (total) { all = total[tid]; before = hist[(int64_t)blockIdx.x * RS_BINS + tid]; }
    else
#pragma unroll 8
        for (int i = 0; i < nblk; ++i) {
            const uint32_t c = hist[(int64_t)i * RS_BINS + tid];
            all += c;
            before += i < (int)blockIdx.x ? c : 0;
        }
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
    const uint32_t first = scan256(all, tot) - all;        // (its barriers: the counts are cleared)
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r)
        if (b + r * 64 < N) atomicAdd(&cnt[wv][(k[r] >> shift) & (RS_BINS - 1)], 1u);
    __syncthreads();
    uint32_t at = first + before;
#pragma unroll
    for (int w = 0; w < 4; ++w) { const uint32_t c = cnt[w][tid]; cnt[w][tid] = at; at += c; }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const bool live = b + r * 64 < N;
        const uint32_t dig = (k[r] >> shift) & (RS_BINS - 1);
        const uint32_t to = digit_place(dig, live, lane, cnt[wv]);
        if (live) {
            key_out[to] = k[r];
            pos_out[to] = ps[r];
        }
    }
}

// Up to RS_SMALL ids: every pass in one workgroup, keys and places in LDS between them -- one launch in place of two a pass (a gradient of 256 ids 23.7 -> 19.0 us,
// of 4096 27.5 -> 22.2).
constexpr int RS_SMALL = 4096, RS_SMALL_THREADS = 1024, RS_SMALL_ROUNDS = RS_SMALL / RS_SMALL_THREADS, RS_SMALL_WAVES = RS_SMALL_THREADS / 64;
__global__ __launch_bounds__(RS_SMALL_THREADS) void rows_sort_small_kernel(const void* ids, int wide, int64_t S, int N, int passes, uint32_t* key_out, uint32_t* pos_out) {
    __shared__ uint32_t key[RS_SMALL], pos[RS_SMALL];
    __shared__ uint32_t cnt[RS_SMALL_WAVES][RS_BINS];
    __shared__ uint32_t tot[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int b = wv * (64 * RS_SMALL_ROUNDS) + lane;
    uint32_t k[RS_SMALL_ROUNDS], ps[RS_SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_SMALL_ROUNDS; ++r) {
        const int n = b + r * 64;
        k[r] = n < N ? row_key(ids, wide, nullptr, S, n) : 0xffffffffu;
        ps[r] = (uint32_t)n;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * RS_BITS;
        for (int i = tid; i < RS_SMALL_WAVES * RS_BINS; i += RS_SMALL_THREADS) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r)
            if (b + r * 64 < N) atomicAdd(&cnt[wv][(k[r] >> shift) & (RS_BINS - 1)], 1u);
        __syncthreads();
        uint32_t all = 0;                      // inclusive over the digits, in the first four wavefronts
        if (tid < RS_BINS) {
            for (int w = 0; w < RS_SMALL_WAVES; ++w) all += cnt[w][tid];
        }
        uint32_t in = all;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(in, o);
            if (lane >= o) in += up;
        }
        if (wv < 4 && lane == 63) tot[wv] = in;
        __syncthreads();
        if (tid < RS_BINS) {
            for (int w = 0; w < wv; ++w) in += tot[w];
            uint32_t at = in - all;
            for (int w = 0; w < RS_SMALL_WAVES; ++w) { const uint32_t c = cnt[w][tid]; cnt[w][tid] = at; at += c; }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r) {
            const bool live = b + r * 64 < N;
            const uint32_t dig = (k[r] >> shift) & (RS_BINS - 1);
            const uint32_t to = digit_place(dig, live, lane, cnt[wv]);
            if (live) { key[to] = k[r]; pos[to] = ps[r]; }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r)
            if (b + r * 64 < N) { k[r] = key[b + r * 64]; ps[r] = pos[b + r * 64]; }
    }
#pragma unroll
    for (int r = 0; r < RS_SMALL_ROUNDS; ++r)
        if (b + r * 64 < N) { key_out[b + r * 64] = k[r]; pos_out[b + r * 64] = ps[r]; }
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

// A launch holds fewer than 2^32 threads along x: workgroups beyond ROW_FOLD go along z.
constexpr int64_t ROW_FOLD = 1 << 22;
__device__ __forceinline__ int64_t row_block() { return blockIdx.x + (int64_t)blockIdx.z * gridDim.x; }
static dim3 row_grid(int64_t n, unsigned across) { return dim3((unsigned)(n < ROW_FOLD ? n : ROW_FOLD), across, (unsigned)((n + ROW_FOLD - 1) / ROW_FOLD)); }

// The sums of the long runs (more than RW_CHUNK places) over one chunk of RW_CHUNK sorted places.  At most two long runs meet a chunk: the one
// of its first place (part[chunk][0]) and the one of its last (part[chunk][1]).  The workgroup's groups take a quarter, a third ... of the places each.
template <typename T, int VEC>
__global__ __launch_bounds__(RW_THREADS) void rows_chunk_kernel(const uint32_t* key, const uint32_t* begin, const uint32_t* pos, const T* dout,
                                                                int64_t ldd, int64_t N, int64_t S, int64_t D, int lanes, typename SeqType<T>::Acc* part) {
    using Acc = typename SeqType<T>::Acc;
    __shared__ Acc lds[RW_THREADS * VEC];
    const RowLane l = row_lane<VEC>(lanes, D);
    const int64_t chunk = row_block(), b = chunk * RW_CHUNK, e = b + RW_CHUNK < N ? b + RW_CHUNK : N;
    if (b >= N) return;
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
            for (int i = 0; i < VEC; ++i) part[(chunk * 2 + slot) * D + l.cb + i] = sum[i];
    }
}

// The runs of more than RW_CHUNK * RW_SUPER places: the partial sums of the chunks of one super chunk, joined the same way
// (T: only the type of the sums matters here).
template <typename Acc, int VEC>
__global__ __launch_bounds__(RW_THREADS) void rows_super_kernel(const uint32_t* key, const uint32_t* begin, int64_t N, int64_t S, int64_t D, int lanes,
                                                                const Acc* part, Acc* super) {
    __shared__ Acc lds[RW_THREADS * VEC];
    const RowLane l = row_lane<VEC>(lanes, D);
    constexpr int64_t PLACES = RW_CHUNK * RW_SUPER;
    const int64_t b = (int64_t)blockIdx.x * PLACES, e = b + PLACES < N ? b + PLACES : N;
    const uint32_t first = key[b], last = key[e - 1];
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t k = slot ? last : first;
        if ((slot && last == first) || k >= S) continue;
        const int64_t rb = begin[k], re = begin[k + 1];
        if (re - rb <= PLACES) continue;
        const int64_t c0 = (rb > b ? rb : b) / RW_CHUNK, m = ((re < e ? re : e) - 1) / RW_CHUNK - c0 + 1;
        const int64_t each = (m + l.R - 1) / l.R, from = l.r * each, to = from + each < m ? from + each : m;
        Acc sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0;
        if (l.live && from < to)
            rows_add<Acc, VEC>(sum, to - from, [&](int64_t i) { return part + ((c0 + from + i) * 2 + ((c0 + from + i) * RW_CHUNK < rb)) * D + l.cb; });
        rows_join<VEC>(sum, lds, l, lanes);
        if (l.live && l.r == 0)
            for (int i = 0; i < VEC; ++i) super[((int64_t)blockIdx.x * 2 + slot) * D + l.cb + i] = sum[i];
    }
}

template <typename T, int VEC, int ROWS>
__global__ __launch_bounds__(RW_THREADS) void rows_sum_kernel(const uint32_t* begin, const uint32_t* pos, const T* dout, int64_t ldd, int64_t S,
                                                              int64_t D, int lanes, double scale, const typename SeqType<T>::Acc* part,
                                                              const typename SeqType<T>::Acc* super, T* grad) {
    using Acc = typename SeqType<T>::Acc;
    __shared__ Acc lds[RW_THREADS * VEC];
    const RowLane l = row_lane<VEC>(lanes, D);
    auto put = [&](int64_t s, const Acc(&sum)[VEC], Acc by) {
        RowVec<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.v[i] = narrow<T>(sum[i] * by);
        row_store(grad + s * D + l.cb, o);
    };
    const int64_t s0 = row_block() * l.R * ROWS;
    if (s0 >= S) return;
    const int rows = l.R * ROWS;
    Acc sum[VEC];
    uint32_t b4[ROWS], e4[ROWS];
    bool is_long = false;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t s = s0 + j * l.R + l.r;
        const bool have = l.r < l.R && s < S;
        b4[j] = have ? begin[s] : 0;
        e4[j] = have ? begin[s + 1] : 0;
        is_long |= e4[j] - b4[j] > RW_CHUNK;
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t s = s0 + j * l.R + l.r;
        if (!l.live || s >= S || e4[j] - b4[j] > RW_CHUNK) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0;
        const uint32_t b = b4[j];
        rows_add<T, VEC>(sum, e4[j] - b, [&](int64_t i) { return dout + (int64_t)pos[b + i] * ldd + l.cb; });
        put(s, sum, e4[j] > b ? (Acc)scale : Acc(0));        // (no id: zero, whatever the scale)
    }
    if (!__syncthreads_or(is_long)) return;
    for (int r = 0; r < rows && s0 + r < S; ++r) {         // the long ones, the whole workgroup at each: partial sums of their chunks
        const int64_t b = begin[s0 + r], e = begin[s0 + r + 1];
        if (e - b <= RW_CHUNK) continue;
        const bool very = super && e - b > RW_CHUNK * RW_SUPER;
        const int64_t places = very ? RW_CHUNK * RW_SUPER : RW_CHUNK;
        const Acc* from_part = very ? super : part;
        const int64_t c0 = b / places, m = (e - 1) / places - c0 + 1;
        const int64_t each = (m + l.R - 1) / l.R, from = l.r * each, to = from + each < m ? from + each : m;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0;
        if (l.live && from < to)
            rows_add<Acc, VEC>(sum, to - from, [&](int64_t i) { return from_part + ((c0 + from + i) * 2 + ((c0 + from + i) * places < b)) * D + l.cb; });
        rows_join<VEC>(sum, lds, l, lanes);
        if (l.live && l.r == 0) put(s0 + r, sum, (Acc)scale);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
struct RowsPlan {
    int nblk, passes;
    int64_t key0, key1, pos0, pos1, hist, total, begin, part, super, bytes;
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
    p.super = take((N + RW_CHUNK * RW_SUPER - 1) / (RW_CHUNK * RW_SUPER) * 2 * D * (type == DCARL_F64 ? 2 : 1));
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
        const int64_t each = (int64_t)(RW_THREADS / lanes) * RW_ROWS, need = (N + each - 1) / each;
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
    if (N > 0 && N <= RS_SMALL) {
        k_in = k_out; p_in = p_out;
        hipLaunchKernelGGL(rows_sort_small_kernel, dim3(1), dim3(RS_SMALL_THREADS), 0, st, ids, id_bytes == 8, S, (int)N, p.passes, k_in, p_in);
    }
    for (int i = 0; i < p.passes && N > RS_SMALL; ++i) {
        const bool direct = p.nblk <= RS_DIRECT;
        hipLaunchKernelGGL(rows_hist_kernel, dim3(p.nblk), dim3(256), 0, st, ids, id_bytes == 8, k_in, S, N, i * RS_BITS, at(p.hist));
        if (!direct) hipLaunchKernelGGL(rows_scan_kernel, dim3(RS_BINS), dim3(256), 0, st, at(p.hist), p.nblk, at(p.total));
        hipLaunchKernelGGL(rows_scatter_kernel, dim3(p.nblk), dim3(256), 0, st, ids, id_bytes == 8, k_in, p_in, S, N, i * RS_BITS, at(p.hist),
                           direct ? nullptr : at(p.total), p.nblk, k_out, p_out);
        k_in = k_out; p_in = p_out;
        k_out = at(i % 2 ? p.key0 : p.key1); p_out = at(i % 2 ? p.pos0 : p.pos1);
    }
    hipLaunchKernelGGL(rows_begin_kernel, dim3((unsigned)((S + 256) / 256)), dim3(256), 0, st, k_in, N, S, at(p.begin));
    rows_with(type, D, [&](auto t, auto V, int lanes, unsigned across) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        Acc *part = reinterpret_cast<Acc*>(w + p.part), *super = reinterpret_cast<Acc*>(w + p.super);
        const int64_t R = RW_THREADS / lanes;
        if (N > RW_CHUNK)
            hipLaunchKernelGGL((rows_chunk_kernel<T, V()>), row_grid((N + RW_CHUNK - 1) / RW_CHUNK, across), dim3(RW_THREADS), 0, st, k_in,
                               at(p.begin), p_in, (const T*)dout, ldd, N, S, D, lanes, part);
        // up to 16384 ids the sums take their chunks one by one (256 at most): a launch less
        if (N <= 8 * RW_CHUNK * RW_SUPER) super = nullptr;
        else
            hipLaunchKernelGGL((rows_super_kernel<Acc, V()>), dim3((unsigned)((N + RW_CHUNK * RW_SUPER - 1) / (RW_CHUNK * RW_SUPER)), across),
                               dim3(RW_THREADS), 0, st, k_in, at(p.begin), N, S, D, lanes, part, super);
        // Four rows per group of threads where that leaves every CU eight workgroups, one otherwise: 50000 rows of 2 KB 22.6 (four) and 36.9 us (one),
        // 8000 rows of 1 KB 43 and 27.
        auto go = [&](auto rows) {
            const int64_t each = R * rows();
            hipLaunchKernelGGL((rows_sum_kernel<T, V(), rows()>), row_grid((S + each - 1) / each, across), dim3(RW_THREADS), 0, st,
                               at(p.begin), p_in, (const T*)dout, ldd, S, D, lanes, scale, part, super, (T*)grad);
        };
        if (S / (R * RW_ROWS) * across >= 2048) go(std::integral_constant<int, RW_ROWS>{});
        else go(std::integral_constant<int, 1>{});
    });
}

}  // namespace dcarl
