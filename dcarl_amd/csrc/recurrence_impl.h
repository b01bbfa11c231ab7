// Gated linear recurrence along ragged episodes: h_t = g_t * h_{t-1} + x_t per channel, restarted from h0[e] (or 0) where episode e
// begins, and its gradients  d_t = dh_t + g_{t+1} d_{t+1},  dx = d,  dg_t = d_t h_{t-1},  dh0[e] = g_s d_s (s: the episode's first step).
//
// A step is the affine map s -> g s + x; the composition of consecutive steps is one again, (A, B) with A the product of the gates, so
// the time axis can be cut anywhere.  Three levels:
//   * a thread walks K consecutive steps of VEC channels held in registers; the 64 / C groups of a wavefront and the four wavefronts of a
//     workgroup hold consecutive segments, so a workgroup takes one tile of 4 * (64 / C) * K steps of C * VEC channels;
//   * the segments' maps are composed by shuffles and through LDS, then each thread walks its steps once more from the state that reaches it;
//   * the state that reaches a tile: every tile publishes its own map as soon as it has it, every group of REC_GROUP tiles its map; a tile joins those
//     between its episode's start and itself, tiles in its own group, whole groups before, and beyond REC_BACK groups the state published there.
//     x and g are read once.
// The waits end: a workgroup takes its tile by a ticket, in time order, so whatever it waits for belongs to workgroups that run already and
// wait in turn only for earlier ones; a wait that takes REC_POLLS polls all the same gives up with NaN
// and says so (rec_gave_up).  A published word is its own flag: the
// words are cleared to a pattern before the launch that no result has (rec_word), written and polled by relaxed atomics of device scope, and
// nothing else passes between workgroups, so no fence is needed.
// An episode's start is a flag, never a gate of zero: what lies before it is dropped, so a NaN there stays there.
// All compositions happen in a fixed order, whoever comes first: run-to-run identical.
// Bound by memory: x, g and h once each (dh, x, g, dx, dg backward), and 8 bytes per channel and tile between workgroups (1 %).  65536 steps of 2048 channels in two
// episodes: bf16 forward 209 us (3.9 TB/s), backward 356 (3.8); 32768 steps in f32 168 (4.8) and 293 (4.6); a copy reaches 5.0 TB/s on the same GPU.  What the 16-bit
// types lack is bytes in flight: a load instruction carries half as many.  Composing the parts' maps in a launch of its own, which reads x and g twice, took
// 322 and 448 us.
#pragma once
#include "seq_common.h"

namespace dcarl {

constexpr int REC_THREADS = 256, REC_WAVES = 4, REC_GROUP = 16, REC_BACK = 4, REC_POLLS = 1 << 20, REC_TICKET = 32;
constexpr int REC_START = 1, REC_END = 2, REC_OUT = 4;     // of a step, in walking order; OUT: behind the last episode

// Step r of the walk is step r, or N - 1 - r for `reverse`: flags, episodes, tiles and maps are in walking order, the operands in their own.
template <typename T> struct RecWalk {
    using Acc = typename SeqType<T>::Acc;
    int64_t N, D, E;
    const int64_t* ep_off;
    int reverse, past, polls;
    int64_t tiles;             // along the time axis
    uint32_t blocks;           // of channels
    const T *x, *g, *h0;
    uint32_t ldx, ldg;
    int64_t ldh0;
    Acc gval;
    const uint8_t* flag;       // [N]
    const int32_t* ep;         // [N]
    const int32_t* from;       // [tiles]: the tile in which the episode that comes into a tile starts; -1: none comes in
    const int32_t* till;       // [tiles]: ... in which the episode that goes on behind it ends; -1: none goes on
    uint32_t* ticket;
    Acc* map;                  // [tiles][lanes][2] (rec_at): the published maps
    Acc* group;                // [tiles / REC_GROUP + 1][lanes][2]: ... of whole groups
    Acc* through;              // [tiles / REC_GROUP + 1][lanes]: the published states that reach the groups
    Acc* state;                // [tiles][D]: the state before each tile (nullable in the forward pass)
    T *h, *last;               // forward: the results
    const T *dh, *dlast;
    uint32_t lddh;
    T *dx, *dg, *dh0;
    Acc* dgp;                  // shared gate: [channel blocks][N] partial sums, or null: one block, straight to dg
};

// K consecutive steps of VEC channels per thread (16-byte loads of f32, 8-byte ones of 16-bit types; 16 steps of those spill).
// One channel alone: 16 (8) steps, side by side in memory, in 16-byte loads -- fewer tiles to hand out and to chain (4e6 steps of one f32 channel: 79 us with
// 8 steps, 52 with 16).
template <typename T, int C> constexpr int REC_K = C == 1 ? (sizeof(T) == 8 ? 8 : 16) : sizeof(T) == 8 ? 4 : 8;
template <typename T> constexpr int REC_VEC = sizeof(T) == 8 ? 2 : 4;

template <typename T, int VEC> struct RecRaw { T v[VEC]; };
// `at` elements behind a workgroup's own base: one scalar address and 32-bit offsets (the host holds TILE * ld to 32 bits).  Rows lie at any multiple of
// the type: unaligned vector accesses.
template <typename T, int VEC> __device__ __forceinline__ RecRaw<T, VEC> rec_load(const T* base, uint32_t at) {
    RecRaw<T, VEC> r;
    __builtin_memcpy(&r, reinterpret_cast<const char*>(base) + (uint32_t)(at * (uint32_t)sizeof(T)), sizeof(r));
    return r;
}
// results that nothing here reads again go past the caches where a workgroup writes whole 128-byte lines (bf16, 65536 steps of 2048 channels: forward 221 -> 207 us,
// backward 354 -> 340); where lines are shared between workgroups the cache joins them (f32, 10007 steps of 999: 30 us, past it 33)
typedef unsigned rec_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned rec_u2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T, int VEC> __device__ __forceinline__ void rec_store(T* base, uint32_t at, const RecRaw<T, VEC>& r, bool past) {
    char* p = reinterpret_cast<char*>(base) + (uint32_t)(at * (uint32_t)sizeof(T));
    if (sizeof(r) < 8 || !past) __builtin_memcpy(p, &r, sizeof(r));
    else if constexpr (sizeof(r) == 16) __builtin_nontemporal_store(__builtin_bit_cast(rec_u4, r), reinterpret_cast<rec_u4*>(p));
    else if constexpr (sizeof(r) == 8) __builtin_nontemporal_store(__builtin_bit_cast(rec_u2, r), reinterpret_cast<rec_u2*>(p));
}

// One channel: a thread's K results side by side, `o` in walking order, those from n on do not exist.
template <typename T, int K> __device__ __forceinline__ void rec_store_row(T* base, int lr, int n, int tile, int reverse, const T (&o)[K], bool past) {
    if (n == K) {
        RecRaw<T, K> v;
#pragma unroll
        for (int k = 0; k < K; ++k) v.v[k] = o[reverse ? K - 1 - k : k];
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < K; i += W) {
            RecRaw<T, W> q;
#pragma unroll
            for (int k = 0; k < W; ++k) q.v[k] = v.v[i + k];
            rec_store(base, (uint32_t)(reverse ? tile - lr - K : lr) + i, q, past);
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < n) base[reverse ? tile - 1 - lr - k : lr + k] = o[k];
    }
}

// a workgroup's tile: the steps row0 .. row0 + rows - 1 of the walk, the first of its rows in memory
struct RecSpan {
    int64_t tile, row0, low;
    int rows;
    uint32_t blk;
};

__device__ __forceinline__ int64_t rec_ep_begin(const int64_t* off, int64_t e, int reverse, int64_t N) {
    const int64_t s = reverse ? N - off[e + 1] : off[e];
    return s < 0 ? 0 : s > N ? N : s;
}
__device__ __forceinline__ int64_t rec_ep_end(const int64_t* off, int64_t e, int reverse, int64_t N) {
    const int64_t s = reverse ? N - off[e] : off[e + 1];
    return s < 0 ? 0 : s > N ? N : s;
}

// the episode around a step, kept while the steps asked for lie in it
struct RecFind {
    int64_t lo = 0, hi = 0, e = -1;                        // steps lo .. hi - 1 of the stream; e < 0: they belong to none
    // flags of step r of the walk
    __device__ __forceinline__ int at(const int64_t* off, int64_t E, int64_t N, int reverse, int64_t r) {
        const int64_t t = reverse ? N - 1 - r : r;
        if (t < lo || t >= hi) {
            int64_t a = 0, b = E + 1;                      // the first offset above t
            while (a < b) {
                const int64_t mid = (a + b) >> 1;
                if (off[mid] <= t) a = mid + 1; else b = mid;
            }
            const bool out = a == 0 || a > E;
            e = out ? -1 : a - 1;
            lo = a == 0 ? 0 : off[a - 1];
            hi = a > E ? N : off[a];
        }
        if (e < 0) return REC_OUT;
        const bool first = t == lo, last = t == hi - 1;
        return ((reverse ? last : first) ? REC_START : 0) | ((reverse ? first : last) ? REC_END : 0);
    }
};

// A call of one tile (short batches) finds its flags itself, in LDS, and saves the launch that finds them for longer ones.
template <int TILE> struct RecOwn {
    uint64_t flag[TILE / 8 + 2];
    int32_t ep[TILE];
};
template <typename T, int TILE> __device__ __forceinline__ void rec_own(const RecWalk<T>& a, RecOwn<TILE>& own) {
    if (a.tiles != 1) return;
    uint8_t* flag = reinterpret_cast<uint8_t*>(own.flag);
    for (int r = threadIdx.x; r < (int)a.N; r += REC_THREADS) {
        RecFind f;
        flag[r] = (uint8_t)f.at(a.ep_off, a.E, a.N, a.reverse, r);
        own.ep[r] = (int32_t)f.e;
    }
    __syncthreads();
}
// (A backward pass reads what the forward one left, which may not have run yet where both are in graphs: an episode of that call, whatever lies there.)
template <typename T, int TILE> __device__ __forceinline__ int32_t rec_ep(const RecWalk<T>& a, const RecOwn<TILE>& own, int64_t r) {
    if (a.tiles == 1) return own.ep[r];
    const int32_t e = a.ep[r];
    return (uint32_t)e < (uint32_t)a.E ? e : 0;
}

// one thread's steps of a tile
template <typename T, int C, int VEC, int GK, bool BACK> struct RecTile {
    using Acc = typename SeqType<T>::Acc;
    static constexpr int K = REC_K<T, C>;
    RecRaw<T, VEC> x[K], g[GK == 2 ? K : 1], dh[BACK ? K : 1];
    T gs[GK == 2 ? 1 : K];
    uint64_t fl[(K + 7) / 8];                              // a byte each
    int n;                                                 // steps that exist
    // K steps of one channel, side by side in memory
    __device__ __forceinline__ static void row(const T* base, uint32_t at, int reverse, RecRaw<T, 1> (&o)[K]) {
        const RecRaw<T, K> v = rec_load<T, K>(base, at);
#pragma unroll
        for (int k = 0; k < K; ++k) o[k].v[0] = reverse ? v.v[K - 1 - k] : v.v[k];
    }
    template <int TILE> __device__ __forceinline__ void flags(const RecWalk<T>& a, const RecSpan& w, const RecOwn<TILE>& own, int lr) {
        const int left = w.rows - lr;
        n = left < 0 ? 0 : left > K ? K : left;
#pragma unroll
        for (int i = 0; i < (K + 7) / 8; ++i) fl[i] = 0;
        if (n > 0) {                                       // (both arrays have K bytes of room behind them)
            if (a.tiles == 1) __builtin_memcpy(fl, reinterpret_cast<const uint8_t*>(own.flag) + lr, K);
            else __builtin_memcpy(fl, a.flag + w.row0 + lr, K);
        }
#pragma unroll
        for (int i = 0; i < (K + 7) / 8; ++i) {
            const int have = n - 8 * i;
            if (have < 8) fl[i] = have <= 0 ? 0 : fl[i] & ((1ull << (8 * have)) - 1);
        }
    }
    // The second walk over the steps widens the 16-bit operands again: without this the compiler keeps the widened ones of the first, in twice the
    // registers (f16 backward, 65536 steps of 2048 channels: 427 us, like this 343).
    __device__ __forceinline__ void again() {
        if constexpr (sizeof(T) == 2 && VEC == 4) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                hide(x[k]);
                if constexpr (GK == 2) hide(g[k]);
                if constexpr (BACK) hide(dh[k]);
            }
        }
    }
    __device__ __forceinline__ static void hide(RecRaw<T, VEC>& r) {
        uint64_t u;
        __builtin_memcpy(&u, &r, sizeof(u));
        asm volatile("" : "+v"(u));
        __builtin_memcpy(&r, &u, sizeof(u));
    }
    // whether all of the thread's steps exist and none is an episode's edge
    __device__ __forceinline__ bool inner() const {
        uint64_t any = 0;
#pragma unroll
        for (int i = 0; i < (K + 7) / 8; ++i) any |= fl[i];
        return any == 0 && n == K;
    }
    // lr: the thread's first step within the tile; at(k): where its k-th lies among the tile's rows in memory
    template <int TILE> __device__ __forceinline__ void load(const RecWalk<T>& a, const RecSpan& w, int lr, uint32_t cb) {
        const T *xb = a.x + w.low * (int64_t)a.ldx, *gb = a.g ? a.g + w.low * (int64_t)a.ldg : nullptr;
        const T* db = BACK ? a.dh + w.low * (int64_t)a.lddh : nullptr;
        if constexpr (C == 1 && VEC == 1) {
            if (a.ldx == 1 && (!a.g || a.ldg == 1) && (!BACK || a.lddh == 1) && lr + K <= w.rows) {
                const uint32_t at = (uint32_t)(a.reverse ? TILE - lr - K : lr);
                row(xb, at, a.reverse, x);
                if constexpr (GK == 2) row(gb, at, a.reverse, g);
                else if (a.g) {
                    RecRaw<T, 1> v[K];
                    row(gb, at, a.reverse, v);
#pragma unroll
                    for (int k = 0; k < K; ++k) gs[k] = v[k].v[0];
                }
                if constexpr (BACK) row(db, at, a.reverse, dh);
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int l = lr + k < w.rows ? lr + k : w.rows - 1;         // steps that do not exist repeat the last
            const uint32_t at = (uint32_t)(a.reverse ? TILE - 1 - l : l);
            x[k] = rec_load<T, VEC>(xb, at * a.ldx + cb);
            if constexpr (GK == 2) g[k] = rec_load<T, VEC>(gb, at * a.ldg + cb);
            else if (a.g) gs[k] = rec_load<T, 1>(gb, at * a.ldg).v[0];
            if constexpr (BACK) dh[k] = rec_load<T, VEC>(db, at * a.lddh + cb);
        }
    }
    __device__ __forceinline__ int flag(int k) const { return (int)(fl[k / 8] >> (8 * (k % 8))) & 7; }
    __device__ __forceinline__ Acc gate(const RecWalk<T>& a, int k, int v) const {
        if constexpr (GK == 2) return widen(g[k].v[v]);
        else return a.g ? widen(gs[k]) : a.gval;
    }
};

// Rows of `base` for those of the thread's steps k0 .. k0 + REC_EDGES - 1 that carry `bit`, zeros for the others; all on the way together (one after
// the other, the rows of one step of 48 episodes took 15 us, like this 9; all K at once spill).
template <typename T> constexpr int REC_EDGES = sizeof(T) == 2 ? 4 : 2;
template <typename T, int VEC> struct RecEdges { RecRaw<T, VEC> v[REC_EDGES<T>]; };
template <typename T, int C, int VEC, int GK, bool BACK, int TILE>
__device__ __forceinline__ void rec_edges(const RecWalk<T>& a, const RecOwn<TILE>& own, const RecTile<T, C, VEC, GK, BACK>& t, int64_t r0, uint32_t cb,
                                          const T* base, int64_t ld, int bit, int k0, RecEdges<T, VEC>& o) {
    int32_t e[REC_EDGES<T>];
#pragma unroll
    for (int k = 0; k < REC_EDGES<T>; ++k) e[k] = base && k0 + k < t.n && (t.flag(k0 + k) & bit) ? rec_ep(a, own, r0 + k0 + k) : -1;
#pragma unroll
    for (int k = 0; k < REC_EDGES<T>; ++k) {
        if (base) __builtin_memcpy(&o.v[k], base + (int64_t)(e[k] < 0 ? 0 : e[k]) * ld + cb, sizeof(o.v[k]));
#pragma unroll
        for (int i = 0; i < VEC; ++i) o.v[k].v[i] = e[k] < 0 ? narrow<T>(0.0f) : o.v[k].v[i];
    }
}

// The map (A, B) at s.  At zero it is B whatever A is: over many steps the product of gates above 1 overflows, and a state of zero stays what the steps make of it.
template <typename Acc> __device__ __forceinline__ Acc rec_apply(Acc A, Acc s, Acc B) {
    const Acc r = fma(A, s, B);
    return s == Acc(0) ? B : r;
}

// (A, B) of a run of steps for VEC channels; `cut`: an episode starts inside, nothing from before comes through
template <typename Acc, int VEC> struct RecMap {
    Acc A[VEC], B[VEC];
    bool cut;
    __device__ __forceinline__ void one() {
#pragma unroll
        for (int v = 0; v < VEC; ++v) { A[v] = 1; B[v] = 0; }
        cut = false;
    }
    // this run after `f`
    __device__ __forceinline__ void after(const RecMap& f) {
        if (cut) return;
#pragma unroll
        for (int v = 0; v < VEC; ++v) { B[v] = rec_apply(A[v], f.B[v], B[v]); A[v] *= f.A[v]; }
        cut = f.cut;
    }
};
template <typename Acc, int VEC> __device__ __forceinline__ RecMap<Acc, VEC> rec_from_lane(const RecMap<Acc, VEC>& m, int lane) {
    RecMap<Acc, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) { o.A[v] = __shfl(m.A[v], lane); o.B[v] = __shfl(m.B[v], lane); }
    o.cut = __shfl((int)m.cut, lane) != 0;
    return o;
}

// The maps of a workgroup's segments are joined in the direction DIR: +1 in time order, -1 against it.  LDS: the wavefronts' totals.
template <typename Acc, int C, int VEC> struct RecShare {
    Acc A[REC_WAVES][C * VEC], B[REC_WAVES][C * VEC];
    int cut[REC_WAVES];
};
// within the wavefront: inclusive scan over the groups; the wavefront's total goes to LDS
template <typename Acc, int C, int VEC, int DIR> __device__ __forceinline__ void rec_scan_groups(RecMap<Acc, VEC>& m, int lane) {
    const int grp = lane / C;
    constexpr int G = 64 / C;
#pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        const RecMap<Acc, VEC> f = rec_from_lane(m, (lane - DIR * o * C) & 63);
        if (DIR > 0 ? grp >= o : grp < G - o) m.after(f);
    }
}
template <typename Acc, int C, int VEC, int DIR>
__device__ __forceinline__ void rec_scan_wave(RecMap<Acc, VEC>& m, RecShare<Acc, C, VEC>& sh, int lane, int wv) {
    const int c = lane % C;
    rec_scan_groups<Acc, C, VEC, DIR>(m, lane);
    if (lane / C == (DIR > 0 ? 64 / C - 1 : 0)) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) { sh.A[wv][c * VEC + v] = m.A[v]; sh.B[wv][c * VEC + v] = m.B[v]; }
        if (c == 0) sh.cut[wv] = m.cut;
    }
}
// after the barrier: `carry` (what reaches the tile) becomes what leaves it, `in` what reaches the thread's segment; m as rec_scan_wave left it
template <typename Acc, int C, int VEC, int DIR>
__device__ __forceinline__ void rec_carry(const RecMap<Acc, VEC>& m, const RecShare<Acc, C, VEC>& sh, int lane, int wv, Acc (&carry)[VEC], Acc (&in)[VEC]) {
    const int c = lane % C, grp = lane / C;
    constexpr int G = 64 / C;
#pragma unroll
    for (int i = 0; i < REC_WAVES; ++i) {
        const int w = DIR > 0 ? i : REC_WAVES - 1 - i;
        if (w == wv) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) in[v] = carry[v];
        }
        const bool cut = sh.cut[w] != 0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc b = sh.B[w][c * VEC + v];
            carry[v] = cut ? b : rec_apply(sh.A[w][c * VEC + v], carry[v], b);
        }
    }
    if constexpr (G > 1) {
        const RecMap<Acc, VEC> f = rec_from_lane(m, (lane - DIR * C) & 63);
        if (DIR > 0 ? grp > 0 : grp < G - 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) in[v] = f.cut ? f.B[v] : rec_apply(f.A[v], in[v], f.B[v]);
        }
    }
}

// the thread's steps as one map, forward in time
template <typename T, int C, int VEC, int GK, bool BACK, int TILE>
__device__ __forceinline__ void rec_map_forward(const RecWalk<T>& a, const RecOwn<TILE>& own, const RecTile<T, C, VEC, GK, BACK>& t, int64_t r0, uint32_t cb,
                                                RecMap<typename SeqType<T>::Acc, VEC>& m) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T, C>;
    m.one();
    if (__all(t.inner())) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Acc g = t.gate(a, k, v);
                m.B[v] = fma(g, m.B[v], (Acc)widen(t.x[k].v[v]));
                m.A[v] *= g;
            }
        return;
    }
    RecEdges<T, VEC> h0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (!BACK)                               // (the backward pass has no registers to spare for them)
            if (k % REC_EDGES<T> == 0) rec_edges(a, own, t, r0, cb, a.h0, a.ldh0, REC_START, k, h0);
        if (k >= t.n) continue;
        const int f = t.flag(k);
        if (f & REC_OUT) { m.cut = true; continue; }
        if (f & REC_START) {
            m.cut = true;
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                m.B[v] = !BACK ? (Acc)widen(h0.v[k % REC_EDGES<T>].v[v]) : a.h0 ? (Acc)widen(a.h0[rec_ep(a, own, r0 + k) * a.ldh0 + cb + v]) : Acc(0);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc g = t.gate(a, k, v);
            m.B[v] = fma(g, m.B[v], (Acc)widen(t.x[k].v[v]));
            m.A[v] *= g;
        }
    }
}
// ... and backward: c -> g (dh + c), from behind; an episode's last step takes dlast instead of what comes from behind it
template <typename T, int C, int VEC, int GK, int TILE>
__device__ __forceinline__ void rec_map_backward(const RecWalk<T>& a, const RecOwn<TILE>& own, const RecTile<T, C, VEC, GK, true>& t, int64_t r0, uint32_t cb,
                                                 RecMap<typename SeqType<T>::Acc, VEC>& m) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T, C>;
    m.one();
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
        if (k >= t.n) continue;
        const int f = t.flag(k);
        if (f & REC_OUT) { m.cut = true; continue; }
        if (f & REC_END) {
            m.cut = true;
#pragma unroll
            for (int v = 0; v < VEC; ++v) m.B[v] = a.dlast ? (Acc)widen(a.dlast[rec_ep(a, own, r0 + k) * a.D + cb + v]) : Acc(0);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc g = t.gate(a, k, v);
            m.B[v] = g * (widen(t.dh[k].v[v]) + m.B[v]);
            m.A[v] *= g;
        }
    }
}

// wavefronts per SIMD: what each instance's registers allow without a spill
template <typename T, int GK> constexpr int REC_WAVES_FORWARD = __is_same(T, float) && GK == 2 ? 3 : 4;
template <typename T, int GK> constexpr int REC_WAVES_BACKWARD = __is_same(T, float) && GK == 2 ? 2 : 3;
template <int C, typename T> constexpr int REC_TILE = REC_WAVES * (64 / C) * REC_K<T, C>;

// ---- between workgroups -----------------------------------------------------------------------------------------------------------------
// a published value as a word that is never the cleared pattern (all ones, a NaN): every NaN is published as the quiet one
__device__ __forceinline__ uint32_t rec_word(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v); }
__device__ __forceinline__ uint64_t rec_word(double v) { return v != v ? 0x7ff8000000000000ull : (uint64_t)__double_as_longlong(v); }
template <typename W> __device__ __forceinline__ void rec_put(W* p, W w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// A wait of this unit's kernels was given up since the host last asked.  (A word per unit and device.)
static __device__ uint32_t rec_gave_up = 0;
static int rec_take() {                  // reads and clears it: 0 or 1, -1 where the device cannot be read
    void* p = nullptr;
    uint32_t v = 0;
    const uint32_t none = 0;
    if (hipGetSymbolAddress(&p, HIP_SYMBOL(rec_gave_up)) != hipSuccess || hipMemcpy(&v, p, sizeof(v), hipMemcpyDeviceToHost) != hipSuccess) return -1;
    if (v && hipMemcpy(p, &none, sizeof(none), hipMemcpyHostToDevice) != hipSuccess) return -1;
    return v != 0;
}
// n words, p(i) the address of the i-th, all in flight together
template <int n, typename W, typename P> __device__ __forceinline__ void rec_poll(W (&w)[n], int polls, P&& p) {
    bool all = false;
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = ~(W)0;
    for (int tries = 0; !all && tries < polls; ++tries) {
        if (tries) __builtin_amdgcn_s_sleep(1);
        all = true;
#pragma unroll
        for (int i = 0; i < n; ++i) w[i] = __hip_atomic_load(p(i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int i = 0; i < n; ++i) all = all && w[i] != (W)~(W)0;
    }
    if (!all) __hip_atomic_store(&rec_gave_up, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);        // what is missing: all ones, a NaN
}
// a map of f32 is one 8-byte word, one of f64 two
__device__ __forceinline__ void rec_put_map(float* p, float A, float B) {
    rec_put(reinterpret_cast<uint64_t*>(p), (uint64_t)rec_word(B) << 32 | rec_word(A));
}
__device__ __forceinline__ void rec_put_map(double* p, double A, double B) {
    rec_put(reinterpret_cast<uint64_t*>(p), rec_word(A));
    rec_put(reinterpret_cast<uint64_t*>(p) + 1, rec_word(B));
}
// maps of VEC channels, p(v) where the v-th lies
template <int VEC, typename P> __device__ __forceinline__ void rec_get_maps(int polls, P&& p, float (&A)[VEC], float (&B)[VEC]) {
    uint64_t w[VEC];
    rec_poll(w, polls, [&](int v) { return reinterpret_cast<const uint64_t*>(p(v)); });
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = __uint_as_float((uint32_t)w[v]); B[v] = __uint_as_float((uint32_t)(w[v] >> 32)); }
}
template <int VEC, typename P> __device__ __forceinline__ void rec_get_maps(int polls, P&& p, double (&A)[VEC], double (&B)[VEC]) {
    uint64_t w[2 * VEC];
    rec_poll(w, polls, [&](int i) { return reinterpret_cast<const uint64_t*>(p(i / 2)) + i % 2; });
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = __longlong_as_double((long long)w[2 * v]); B[v] = __longlong_as_double((long long)w[2 * v + 1]); }
}
__device__ __forceinline__ void rec_put_state(float* p, float v) { rec_put(reinterpret_cast<uint32_t*>(p), rec_word(v)); }
__device__ __forceinline__ void rec_put_state(double* p, double v) { rec_put(reinterpret_cast<uint64_t*>(p), rec_word(v)); }
template <int VEC, typename P> __device__ __forceinline__ void rec_get_states(int polls, P&& p, float (&s)[VEC]) {
    uint32_t w[VEC];
    rec_poll(w, polls, [&](int v) { return reinterpret_cast<const uint32_t*>(p(v)); });
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = __uint_as_float(w[v]);
}
template <int VEC, typename P> __device__ __forceinline__ void rec_get_states(int polls, P&& p, double (&s)[VEC]) {
    uint64_t w[VEC];
    rec_poll(w, polls, [&](int v) { return reinterpret_cast<const uint64_t*>(p(v)); });
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = __longlong_as_double((long long)w[v]);
}

// The tile's number in time order within its block of channels.  A counter per block, since chains of two blocks do not meet: one for all took the longest
// forward pass from 271 to 285 us.  (It still hands out some 20 ns apart, which is what long streams of few channels are bound by.)
template <typename T> __device__ __forceinline__ RecSpan rec_span(const RecWalk<T>& a, int tile_rows, bool back) {
    RecSpan w;
    w.blk = blockIdx.x % a.blocks;
    w.tile = 0;
    if (a.tiles > 1) {
        __shared__ uint32_t mine;
        if (threadIdx.x == 0) mine = atomicAdd(a.ticket + w.blk * REC_TICKET, 1u);
        __syncthreads();
        w.tile = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine);
    }
    if (back) w.tile = a.tiles - 1 - w.tile;
    w.row0 = w.tile * tile_rows;
    w.rows = (int)(a.N - w.row0 < tile_rows ? a.N - w.row0 : tile_rows);
    w.low = a.reverse ? a.N - w.row0 - tile_rows : w.row0;
    return w;
}

// the whole tile's map, from the wavefronts' totals
template <typename Acc, int C, int VEC, int DIR>
__device__ __forceinline__ RecMap<Acc, VEC> rec_total(const RecShare<Acc, C, VEC>& sh, int c) {
    RecMap<Acc, VEC> t;
    t.one();
#pragma unroll
    for (int i = 0; i < REC_WAVES; ++i) {
        const int w = DIR > 0 ? i : REC_WAVES - 1 - i;
        RecMap<Acc, VEC> m;
        m.cut = sh.cut[w] != 0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) { m.A[v] = sh.A[w][c * VEC + v]; m.B[v] = sh.B[w][c * VEC + v]; }
        m.after(t);
        t = m;
    }
    return t;
}

// Where the v-th word of lane c lies among those of tile (group) n: the lanes side by side, so that a wavefront's access is a few whole lines (channel by
// channel, 8 bytes every 32, the longest forward pass took 290 us, like this 251).
template <int C, int VEC> __device__ __forceinline__ int64_t rec_at(int64_t n, uint32_t blocks, uint32_t blk, int v, int c) {
    return ((n * blocks + blk) * VEC + v) * C + c;
}

// What reaches `tile` of an episode that comes in from the tile `from` (DIR > 0: an earlier one; < 0: a later one):
//   P, the map of the tiles of its own group between `from` and itself: the thread group j takes the map of tile j of the group, as if it were a segment of
//   its own, and they are joined as segments are; `from` itself passes on its B alone;
//   the state that reaches the group: the maps of the up to REC_BACK groups before, on what reaches the first of them -- published REC_BACK groups ago, so
//   that the chain of a longer episode has one link per REC_BACK groups (262144 steps of 64 channels in one episode: 87 us with a link per group, 53 like this;
//   streams of many channels do not notice).
// The group's last tile publishes the group's map before it waits for that state, and then what leaves the group.
template <typename T, int C, int VEC, int DIR>
__device__ __forceinline__ void rec_reach(const RecWalk<T>& a, int64_t tile, int from, uint32_t blk, int lane, int wv, bool mine,
                                          const RecMap<typename SeqType<T>::Acc, VEC>& total, RecShare<typename SeqType<T>::Acc, C, VEC>& sh,
                                          typename SeqType<T>::Acc (&reached)[C * VEC], typename SeqType<T>::Acc (&carry)[VEC]) {
    using Acc = typename SeqType<T>::Acc;
    const int64_t group = tile / REC_GROUP;
    const bool closes = DIR > 0 ? tile % REC_GROUP == REC_GROUP - 1 && tile + 1 < a.tiles : tile % REC_GROUP == 0 && tile > 0;
    const int c = lane % C, j = wv * (64 / C) + lane / C;
    const bool first = wv == 0 && lane < C && mine;        // the threads that publish
    auto at = [&](int64_t n, int v) { return rec_at<C, VEC>(n, a.blocks, blk, v, c); };
    const int64_t src = group * REC_GROUP + j;
    RecMap<Acc, VEC> m;
    m.one();
    if (from >= 0) {                                       // (otherwise an episode starts with the tile: its map is all there is)
        if (j < REC_GROUP && mine && (DIR > 0 ? src < tile && src >= from : src > tile && src <= from)) {
            rec_get_maps<VEC>(a.polls, [&](int v) { return a.map + at(src, v) * 2; }, m.A, m.B);
            m.cut = src == from;
        }
        rec_scan_wave<Acc, C, VEC, DIR>(m, sh, lane, wv);
        __syncthreads();
        m = rec_total<Acc, C, VEC, DIR>(sh, c);            // P
    }
    const bool outside = from >= 0 && (DIR > 0 ? from < group * REC_GROUP : from >= (group + 1) * REC_GROUP);
    if (closes && first) {
        RecMap<Acc, VEC> g = total;
        g.after(m);
#pragma unroll
        for (int v = 0; v < VEC; ++v) rec_put_map(a.group + at(group, v) * 2, g.A[v], g.B[v]);
    }
    if (outside) {
        if (wv == 0) {
            // the groups fg .. group - 1 (DIR > 0), at most the last REC_BACK of them, a thread group each; fg itself passes on its B alone
            const int64_t fg = from / REC_GROUP, far = group - DIR * REC_BACK;
            const bool chain = DIR > 0 ? fg < far : fg > far;
            const int64_t g = DIR > 0 ? (chain ? far : fg) + lane / C : group + 1 + lane / C;
            RecMap<Acc, VEC> q;
            q.one();
            if (mine && (DIR > 0 ? g < group : g <= (chain ? far : fg))) {
                rec_get_maps<VEC>(a.polls, [&](int v) { return a.group + at(g, v) * 2; }, q.A, q.B);
                q.cut = g == fg;
            }
            rec_scan_groups<Acc, C, VEC, DIR>(q, lane);
            if (mine && lane / C == (DIR > 0 ? 64 / C - 1 : 0)) {
                Acc st[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) st[v] = 0;
                if (chain) rec_get_states<VEC>(a.polls, [&](int v) { return a.through + at(far, v); }, st);
#pragma unroll
                for (int v = 0; v < VEC; ++v) reached[c * VEC + v] = q.cut ? q.B[v] : rec_apply(q.A[v], st[v], q.B[v]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = from < 0 ? Acc(0) : m.cut ? m.B[v] : rec_apply(m.A[v], outside ? reached[c * VEC + v] : Acc(0), m.B[v]);
    if (closes && first)                                   // what reaches the next group
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            rec_put_state(a.through + at(group + DIR, v), total.cut ? total.B[v] : rec_apply(total.A[v], carry[v], total.B[v]));
}

template <typename T, int C, int VEC, int GK>
__global__ __launch_bounds__(REC_THREADS, (REC_WAVES_FORWARD<T, GK>)) void rec_forward_kernel(RecWalk<T> a) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T, C>, TILE = REC_TILE<C, T>;
    __shared__ RecShare<Acc, C, VEC> share, reach;
    __shared__ RecOwn<TILE> own;
    __shared__ Acc reached[C * VEC];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane % C;
    if (blockIdx.x >= a.tiles * a.blocks) {                                 // the states that empty episodes end with
        const int64_t groups = REC_THREADS / 64, first = (blockIdx.x - a.tiles * a.blocks) * groups + wv, step = ((int64_t)gridDim.x - a.tiles * a.blocks) * groups;
        for (int64_t e = first; e < a.E; e += step)
            if (rec_ep_begin(a.ep_off, e, a.reverse, a.N) >= rec_ep_end(a.ep_off, e, a.reverse, a.N))
                for (int64_t d = lane; d < a.D; d += 64) a.last[e * a.D + d] = a.h0 ? a.h0[e * a.ldh0 + d] : narrow<T>(0.0f);
        return;
    }
    const RecSpan w = rec_span(a, TILE, false);
    const int64_t tile = w.tile;
    const int from = a.tiles > 1 ? a.from[tile] : -1;
    const int64_t c0 = ((int64_t)w.blk * C + c) * VEC;
    const bool mine = c0 < a.D;
    const uint32_t cb = (uint32_t)(c0 < a.D - VEC ? c0 : a.D - VEC);     // the last lanes move back to whole vectors: the same channels, the same values
    const int lr = (wv * (64 / C) + lane / C) * K;
    const int64_t r0 = w.row0 + lr;
    RecTile<T, C, VEC, GK, false> t;
    t.template load<TILE>(a, w, lr, cb);                   // (on the way while a call of one tile finds its flags)
    rec_own(a, own);
    t.flags(a, w, own, lr);
    RecMap<Acc, VEC> m;
    rec_map_forward(a, own, t, r0, cb, m);
    rec_scan_wave<Acc, C, VEC, 1>(m, share, lane, wv);
    __syncthreads();
    const bool first = wv == 0 && lane < C && mine;        // the threads that publish
    Acc carry[VEC], s[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = 0;
    if (a.tiles > 1) {
        const RecMap<Acc, VEC> total = rec_total<Acc, C, VEC, 1>(share, c);
        if (first && tile + 1 < a.tiles)
#pragma unroll
            for (int v = 0; v < VEC; ++v) rec_put_map(a.map + rec_at<C, VEC>(tile, a.blocks, w.blk, v, c) * 2, total.A[v], total.B[v]);
        rec_reach<T, C, VEC, 1>(a, tile, from, w.blk, lane, wv, mine, total, reach, reached, carry);
    }
    if (a.state && first)
        for (int v = 0; v < VEC; ++v) a.state[tile * a.D + cb + v] = carry[v];
    rec_carry<Acc, C, VEC, 1>(m, share, lane, wv, carry, s);
    t.again();
    const bool plain = __all(t.inner());
    T* hb = a.h + w.low * a.D;
    RecEdges<T, VEC> h0;
    T line[C == 1 ? K : 1];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!plain) {
            if (k % REC_EDGES<T> == 0) rec_edges(a, own, t, r0, cb, a.h0, a.ldh0, REC_START, k, h0);
            if (k >= t.n) continue;
            if (t.flag(k) & REC_START) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) s[v] = widen(h0.v[k % REC_EDGES<T>].v[v]);
            }
        }
        RecRaw<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            s[v] = fma(t.gate(a, k, v), s[v], (Acc)widen(t.x[k].v[v]));
            o.v[v] = narrow<T>(s[v]);
        }
        if (!plain && (t.flag(k) & REC_OUT)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) { s[v] = 0; o.v[v] = narrow<T>(0.0f); }
        }
        if constexpr (C == 1) line[k] = o.v[0];
        if (mine) {
            if constexpr (C > 1) rec_store(hb, (uint32_t)(a.reverse ? TILE - 1 - lr - k : lr + k) * (uint32_t)a.D + cb, o, a.past);
            if (a.last && !plain && (t.flag(k) & REC_END)) __builtin_memcpy(a.last + rec_ep(a, own, r0 + k) * a.D + cb, &o, sizeof(o));
        }
    }
    if constexpr (C == 1) rec_store_row<T, K>(hb, lr, t.n, TILE, a.reverse, line, a.past);
}

template <typename T, int C, int VEC, int GK>
__global__ __launch_bounds__(REC_THREADS, (REC_WAVES_BACKWARD<T, GK>)) void rec_backward_kernel(RecWalk<T> a) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T, C>, TILE = REC_TILE<C, T>;
    __shared__ RecShare<Acc, C, VEC> share_b, share_f, reach;
    __shared__ RecOwn<TILE> own;
    __shared__ Acc reached[C * VEC];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane % C;
    if (blockIdx.x >= a.tiles * a.blocks) {                                // an empty episode hands its dlast through
        const int64_t groups = REC_THREADS / 64, first = (blockIdx.x - a.tiles * a.blocks) * groups + wv, step = ((int64_t)gridDim.x - a.tiles * a.blocks) * groups;
        for (int64_t e = first; e < a.E; e += step)
            if (rec_ep_begin(a.ep_off, e, a.reverse, a.N) >= rec_ep_end(a.ep_off, e, a.reverse, a.N))
                for (int64_t d = lane; d < a.D; d += 64) a.dh0[e * a.D + d] = a.dlast ? a.dlast[e * a.D + d] : narrow<T>(0.0f);
        return;
    }
    const RecSpan w = rec_span(a, TILE, true);             // from the end of time
    const int64_t tile = w.tile;
    int till = a.tiles > 1 ? a.till[tile] : -1;
    if (till >= a.tiles) till = (int)a.tiles - 1;          // (as rec_ep: a tile that publishes, whatever lies there)
    const int64_t c0 = ((int64_t)w.blk * C + c) * VEC;
    const bool mine = c0 < a.D;
    const uint32_t cb = (uint32_t)(c0 < a.D - VEC ? c0 : a.D - VEC);
    const int lr = (wv * (64 / C) + lane / C) * K;
    const int64_t r0 = w.row0 + lr;
    RecTile<T, C, VEC, GK, true> t;
    t.template load<TILE>(a, w, lr, cb);                   // (on the way while a call of one tile finds its flags)
    rec_own(a, own);
    t.flags(a, w, own, lr);
    Acc state[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) state[v] = a.state[tile * a.D + cb + v];
    RecMap<Acc, VEC> mb, mf;
    rec_map_backward(a, own, t, r0, cb, mb);
    rec_scan_wave<Acc, C, VEC, -1>(mb, share_b, lane, wv);
    rec_map_forward(a, own, t, r0, cb, mf);
    rec_scan_wave<Acc, C, VEC, 1>(mf, share_f, lane, wv);
    __syncthreads();
    const bool first = wv == 0 && lane < C && mine;
    Acc carry[VEC], s[VEC], back[VEC], prev[K][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = 0;
    if (a.tiles > 1) {
        const RecMap<Acc, VEC> total = rec_total<Acc, C, VEC, -1>(share_b, c);
        if (first && tile > 0)
#pragma unroll
            for (int v = 0; v < VEC; ++v) rec_put_map(a.map + rec_at<C, VEC>(tile, a.blocks, w.blk, v, c) * 2, total.A[v], total.B[v]);
        rec_reach<T, C, VEC, -1>(a, tile, till, w.blk, lane, wv, mine, total, reach, reached, carry);
    }
    rec_carry<Acc, C, VEC, -1>(mb, share_b, lane, wv, carry, back);
    rec_carry<Acc, C, VEC, 1>(mf, share_f, lane, wv, state, s);
    t.again();
#pragma unroll
    for (int k = 0; k < K; ++k) {                          // the states before each step once more, in 32 bits
        if (k < t.n && (t.flag(k) & REC_START)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = a.h0 ? (Acc)widen(a.h0[rec_ep(a, own, r0 + k) * a.ldh0 + cb + v]) : Acc(0);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            prev[k][v] = s[v];
            s[v] = fma(t.gate(a, k, v), s[v], (Acc)widen(t.x[k].v[v]));
        }
    }
    Acc sum[K];
    T line_x[C == 1 ? K : 1], line_g[C == 1 ? K : 1];
    T *dxb = a.dx + w.low * a.D, *dgb = a.dg + (GK == 2 ? w.low * a.D : w.low);
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
        sum[k] = 0;
        if (k >= t.n) continue;
        const int f = t.flag(k);
        if (f & REC_END) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) back[v] = a.dlast ? (Acc)widen(a.dlast[rec_ep(a, own, r0 + k) * a.D + cb + v]) : Acc(0);
        }
        RecRaw<T, VEC> ox, og;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc d = widen(t.dh[k].v[v]) + back[v], term = d * prev[k][v];
            ox.v[v] = narrow<T>(d);
            og.v[v] = narrow<T>(term);
            if (GK == 1 && cb + v >= c0 && !(f & REC_OUT)) sum[k] += term;       // a channel counts in one lane only
            back[v] = t.gate(a, k, v) * d;
        }
        if (f & REC_OUT) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) { ox.v[v] = og.v[v] = narrow<T>(0.0f); back[v] = 0; }
        }
        if constexpr (C == 1) { line_x[k] = ox.v[0]; line_g[k] = og.v[0]; }
        if (mine) {
            const uint32_t at = (uint32_t)(a.reverse ? TILE - 1 - lr - k : lr + k) * (uint32_t)a.D + cb;
            if (C > 1 && a.dx) rec_store(dxb, at, ox, a.past);
            if (C > 1 && GK == 2 && a.dg) rec_store(dgb, at, og, a.past);
            if (a.dh0 && (f & REC_START)) {
                RecRaw<T, VEC> o0;
#pragma unroll
                for (int v = 0; v < VEC; ++v) o0.v[v] = narrow<T>(back[v]);
                __builtin_memcpy(a.dh0 + rec_ep(a, own, r0 + k) * a.D + cb, &o0, sizeof(o0));
            }
        }
    }
    if constexpr (C == 1) {
        if (a.dx) rec_store_row<T, K>(dxb, lr, t.n, TILE, a.reverse, line_x, a.past);
        if (GK == 2 && a.dg) rec_store_row<T, K>(dgb, lr, t.n, TILE, a.reverse, line_g, a.past);
    }
    if constexpr (GK == 1) {
        if (a.dg) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                Acc v = mine ? sum[k] : Acc(0);
#pragma unroll
                for (int o = 1; o < C; o <<= 1) v += __shfl_xor(v, o);
                if (c == 0 && k < t.n) {
                    if (a.dgp) a.dgp[(int64_t)w.blk * a.N + r0 + k] = v;
                    else dgb[a.reverse ? TILE - 1 - lr - k : lr + k] = narrow<T>(v);
                }
            }
        }
    }
}

// f(C, VEC) for the number of channels: one lane per step and channel for few, else vectors; wide rows in 128-byte pieces of a 16-bit type
template <typename T, typename F> inline void rec_with_shape(int64_t D, F&& f) {
    constexpr int V = REC_VEC<T>;
    if (D == 1) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    else if (D < 8) f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    else if (D <= 4 * V) f(std::integral_constant<int, 4>{}, std::integral_constant<int, V>{});
    else f(std::integral_constant<int, 16>{}, std::integral_constant<int, V>{});
}

// workgroups that look for empty episodes, beside those of the tiles
inline unsigned rec_empty_blocks(bool wanted, int64_t E) { return wanted ? (unsigned)((E + 1023) / 1024 < 1024 ? (E + 1023) / 1024 : 1024) : 0; }

struct RecPlan {
    int tile;
    int64_t tiles, blocks, wide;                           // wide: channels of all blocks' lanes
    int64_t flag, ep, from, till, plan_bytes;                          // the walk: in the states where there are any, else in the workspace
    int64_t state, states_bytes;
    int64_t ticket, map, group, through, clear_bytes;             // what passes between workgroups: cleared before each launch
    int64_t dgp, ws_plan, ws_bytes;
};
RecPlan rec_plan(int64_t N, int64_t D, int type, int gate_kind);

int recurrence_status_backward();
template <typename T> void rec_launch_forward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st);
template <typename T> void rec_launch_backward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st);

}  // namespace dcarl
