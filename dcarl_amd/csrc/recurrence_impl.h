// Gated linear recurrence along ragged episodes: h_t = g_t * h_{t-1} + x_t per channel, restarted from h0[e] (or 0) where episode e
// begins, and its gradients  d_t = dh_t + g_{t+1} d_{t+1},  dx = d,  dg_t = d_t h_{t-1},  dh0[e] = g_s d_s (s: the episode's first step).
//
// A step is the affine map s -> g s + x; the composition of consecutive steps is one again, (A, B) with A the product of the gates, so
// the time axis can be cut anywhere.  Three levels:
//   * a thread walks K consecutive steps of VEC channels held in registers; the 64 / C groups of a wavefront and the four wavefronts of a
//     workgroup hold consecutive segments, so a workgroup takes a tile of 4 * (64 / C) * K steps of C * VEC channels at a time: the
//     segments' maps are composed by shuffles and through LDS (one barrier per tile), then each thread walks its steps once more
//     from the state that reaches it.  x and g are read once; the next tile is in flight meanwhile.
//   * a workgroup walks its part of the time axis tile by tile, the state in registers.
//   * where channels alone do not fill the GPU the axis is cut into parts; a first launch composes the maps of the parts whose last episode
//     goes on in the next one (from that episode's start: the others end early), and a part folds those of the parts before it.  The cuts
//     are moved to the nearest episode start within a quarter of a part, which spares that reading where episodes are short.
// An episode's start is a flag, never a gate of zero: what lies before it is dropped, so a NaN there stays there.
// All compositions happen in a fixed order: run-to-run identical.
#pragma once
#include "seq_common.h"

namespace dcarl {

constexpr int REC_THREADS = 256, REC_WAVES = 4, REC_MAX_PARTS = 256;
constexpr int REC_START = 1, REC_END = 2, REC_OUT = 4;     // of a step, in walking order; OUT: behind the last episode

// everything in walking order: step r of the walk is step r, or N - 1 - r for `reverse` (base addresses and strides say so)
template <typename T> struct RecWalk {
    using Acc = typename SeqType<T>::Acc;
    int64_t N, D, E;
    const int64_t* ep_off;
    int reverse, P;
    const T *x, *g, *h0;
    int64_t sx, sg, ldh0;
    Acc gval;
    const uint8_t* flag;       // [N]
    const int32_t* ep;         // [N]
    const int64_t* part;       // [P + 1]
    Acc* agg;                  // [P][2][D]: the maps of the parts
    Acc* state;                // [slots][D]: the state before each tile (nullable in the forward pass)
    T* h; int64_t sh;          // forward: the result
    T* last;
    const T *dh, *dlast; int64_t sdh;
    T *dx, *dg, *dh0;          // sh is their stride, too (dg of a shared gate: 1 or -1)
    Acc* dgp;                  // shared gate: [channel blocks][N] partial sums, or null: one block, straight to dg
};

// K consecutive steps (16-byte loads of f32, 8-byte ones of 16-bit types; registers allow twice the steps of the narrow types)
template <typename T> constexpr int REC_K = sizeof(T) == 2 ? 8 : 4;
template <typename T> constexpr int REC_VEC = sizeof(T) == 8 ? 2 : 4;

template <typename T, int VEC> struct RecRaw { T v[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ RecRaw<T, VEC> rec_load(const T* p) {
    RecRaw<T, VEC> r;
    __builtin_memcpy(&r, p, sizeof(r));                    // rows lie at any multiple of the type: an unaligned vector load
    return r;
}

__device__ __forceinline__ int64_t rec_ep_begin(const int64_t* off, int64_t e, int reverse, int64_t N) {
    const int64_t s = reverse ? N - off[e + 1] : off[e];
    return s < 0 ? 0 : s > N ? N : s;
}
__device__ __forceinline__ int64_t rec_ep_end(const int64_t* off, int64_t e, int reverse, int64_t N) {
    const int64_t s = reverse ? N - off[e] : off[e + 1];
    return s < 0 ? 0 : s > N ? N : s;
}

// one thread's steps of a tile
template <typename T, int C, int VEC, int GK, bool BACK> struct RecTile {
    using Acc = typename SeqType<T>::Acc;
    static constexpr int K = REC_K<T>;
    RecRaw<T, VEC> x[K], g[GK == 2 ? K : 1], dh[BACK ? K : 1];
    T gs[GK == 2 ? 1 : K];
    uint64_t fl;
    int n;                                                 // steps that exist
    __device__ __forceinline__ void load(const RecWalk<T>& a, int64_t r0, int64_t row1, int64_t cb, bool want_x) {
        const int64_t left = row1 - r0;
        n = left < 0 ? 0 : left > K ? K : (int)left;
        fl = 0;
        if (n > 0) __builtin_memcpy(&fl, a.flag + r0, K);  // the array has K bytes of room behind it
        if (n < K) fl = n <= 0 ? 0 : fl & ((1ull << (8 * n)) - 1);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int64_t r = r0 + k;
            r = r < row1 ? r : row1 - 1;
            if (want_x) x[k] = rec_load<T, VEC>(a.x + r * a.sx + cb);
            if constexpr (GK == 2) g[k] = rec_load<T, VEC>(a.g + r * a.sg + cb);
            else if (a.g) gs[k] = a.g[r * a.sg];
            if constexpr (BACK) dh[k] = rec_load<T, VEC>(a.dh + r * a.sdh + cb);
        }
    }
    __device__ __forceinline__ int flag(int k) const { return (int)(fl >> (8 * k)) & 7; }
    __device__ __forceinline__ Acc gate(const RecWalk<T>& a, int k, int v) const {
        if constexpr (GK == 2) return widen(g[k].v[v]);
        else return a.g ? widen(gs[k]) : a.gval;
    }
};

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
        for (int v = 0; v < VEC; ++v) { B[v] = fma(A[v], f.B[v], B[v]); A[v] *= f.A[v]; }
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

// the maps of a workgroup's segments, in `dir` = +1 (time order) or -1: the carry that reaches this thread's segment, the carry behind the
// tile (both from `carry` before it).  m: the thread's own map, overwritten.  LDS: [WAVES][C * VEC] maps.
template <typename Acc, int C, int VEC> struct RecShare {
    Acc A[REC_WAVES][C * VEC], B[REC_WAVES][C * VEC];
    int cut[REC_WAVES];
};
// within the wavefront: inclusive scan over the groups; the wavefront's total goes to LDS
template <typename Acc, int C, int VEC, int DIR>
__device__ __forceinline__ void rec_scan_wave(RecMap<Acc, VEC>& m, RecShare<Acc, C, VEC>& sh, int lane, int wv) {
    const int c = lane % C, grp = lane / C;
    constexpr int G = 64 / C;
#pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        const RecMap<Acc, VEC> f = rec_from_lane(m, (lane - DIR * o * C) & 63);
        if (DIR > 0 ? grp >= o : grp < G - o) m.after(f);
    }
    if (grp == (DIR > 0 ? G - 1 : 0)) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) { sh.A[wv][c * VEC + v] = m.A[v]; sh.B[wv][c * VEC + v] = m.B[v]; }
        if (c == 0) sh.cut[wv] = m.cut;
    }
}
// after the barrier: `carry` (what reaches the tile) becomes what leaves it; returns what reaches the thread's segment
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
            carry[v] = cut ? b : fma(sh.A[w][c * VEC + v], carry[v], b);
        }
    }
    if constexpr (G > 1) {
        const RecMap<Acc, VEC> f = rec_from_lane(m, (lane - DIR * C) & 63);
        if (DIR > 0 ? grp > 0 : grp < G - 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) in[v] = f.cut ? f.B[v] : fma(f.A[v], in[v], f.B[v]);
        }
    }
}

// the thread's steps as one map, forward in time
template <typename T, int C, int VEC, int GK, bool BACK>
__device__ __forceinline__ void rec_map_forward(const RecWalk<T>& a, const RecTile<T, C, VEC, GK, BACK>& t, int64_t r0, int64_t cb,
                                                RecMap<typename SeqType<T>::Acc, VEC>& m) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T>;
    m.one();
    if (__all(t.fl == 0 && t.n == K)) {
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
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (k >= t.n) continue;
        const int f = t.flag(k);
        if (f & REC_OUT) { m.cut = true; continue; }
        if (f & REC_START) {
            m.cut = true;
#pragma unroll
            for (int v = 0; v < VEC; ++v) m.B[v] = a.h0 ? (Acc)widen(a.h0[a.ep[r0 + k] * a.ldh0 + cb + v]) : Acc(0);
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
template <typename T, int C, int VEC, int GK>
__device__ __forceinline__ void rec_map_backward(const RecWalk<T>& a, const RecTile<T, C, VEC, GK, true>& t, int64_t r0, int64_t cb,
                                                 RecMap<typename SeqType<T>::Acc, VEC>& m) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T>;
    m.one();
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
        if (k >= t.n) continue;
        const int f = t.flag(k);
        if (f & REC_OUT) { m.cut = true; continue; }
        if (f & REC_END) {
            m.cut = true;
#pragma unroll
            for (int v = 0; v < VEC; ++v) m.B[v] = a.dlast ? (Acc)widen(a.dlast[a.ep[r0 + k] * a.D + cb + v]) : Acc(0);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc g = t.gate(a, k, v);
            m.B[v] = g * (widen(t.dh[k].v[v]) + m.B[v]);
            m.A[v] *= g;
        }
    }
}

template <int C, typename T> constexpr int REC_TILE = REC_WAVES * (64 / C) * REC_K<T>;

template <typename T, int C, int VEC, int GK, bool AGG>
__global__ __launch_bounds__(REC_THREADS) void rec_forward_kernel(RecWalk<T> a) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T>, TILE = REC_TILE<C, T>;
    __shared__ RecShare<Acc, C, VEC> share[2];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane % C;
    const int64_t c0 = ((int64_t)blockIdx.x * C + c) * VEC;
    const bool mine = c0 < a.D;
    const int64_t cb = c0 < a.D - VEC ? c0 : a.D - VEC;    // the last lanes move back to whole vectors: the same channels, the same values
    if (!AGG && (int)blockIdx.y >= a.P) {                  // the states that empty episodes end with
        const int64_t step = (int64_t)(gridDim.y - a.P) * REC_WAVES * (64 / C);
        for (int64_t e = (((int64_t)blockIdx.y - a.P) * REC_WAVES + wv) * (64 / C) + lane / C; e < a.E; e += step)
            if (rec_ep_begin(a.ep_off, e, a.reverse, a.N) >= rec_ep_end(a.ep_off, e, a.reverse, a.N) && mine)
                for (int v = 0; v < VEC; ++v) a.last[e * a.D + cb + v] = a.h0 ? a.h0[e * a.ldh0 + cb + v] : narrow<T>(0.0f);
        return;
    }
    const int p = blockIdx.y;
    int64_t row0 = a.part[p];
    const int64_t row1 = a.part[p + 1];
    if (row0 >= row1) return;
    int64_t slot = row0 / TILE + p;
    Acc carry[VEC];
    RecMap<Acc, VEC> whole;
    if constexpr (AGG) {
        if (row1 >= a.N || (a.flag[row1] & (REC_START | REC_OUT))) return;         // no episode goes on behind this part
        const int64_t s = rec_ep_begin(a.ep_off, a.ep[row1], a.reverse, a.N);
        row0 = s > row0 && s < row1 ? s : row0;
        whole.one();
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) carry[v] = 0;
        if (p > 0 && !(a.flag[row0] & (REC_START | REC_OUT))) {
            const int64_t s = rec_ep_begin(a.ep_off, a.ep[row0], a.reverse, a.N);
            int q = p - 1;
            while (q > 0 && a.part[q] > s) --q;
            for (bool first = true; q < p; ++q, first = false) {
                if (a.part[q] >= a.part[q + 1]) continue;
                const Acc* m = a.agg + (int64_t)q * 2 * a.D + cb;
#pragma unroll
                for (int v = 0; v < VEC; ++v) carry[v] = first ? m[a.D + v] : fma(m[v], carry[v], m[a.D + v]);
            }
        }
    }
    const int64_t seg = (int64_t)(wv * (64 / C) + lane / C) * K;
    RecTile<T, C, VEC, GK, false> t, next;
    t.load(a, row0 + seg, row1, cb, true);
    int buf = 0;
    for (int64_t base = row0; base < row1; base += TILE, buf ^= 1, ++slot) {
        if (base + TILE < row1) next.load(a, base + TILE + seg, row1, cb, true);
        const int64_t r0 = base + seg;
        RecMap<Acc, VEC> m;
        rec_map_forward(a, t, r0, cb, m);
        rec_scan_wave<Acc, C, VEC, 1>(m, share[buf], lane, wv);
        __syncthreads();
        if constexpr (AGG) {
#pragma unroll
            for (int w = 0; w < REC_WAVES; ++w) {
                RecMap<Acc, VEC> f = whole;
                whole.cut = share[buf].cut[w] != 0;
#pragma unroll
                for (int v = 0; v < VEC; ++v) { whole.A[v] = share[buf].A[w][c * VEC + v]; whole.B[v] = share[buf].B[w][c * VEC + v]; }
                whole.after(f);
            }
        } else {
            Acc s[VEC];
            if (a.state && mine && wv == 0 && lane < C)
                for (int v = 0; v < VEC; ++v) a.state[slot * a.D + cb + v] = carry[v];
            rec_carry<Acc, C, VEC, 1>(m, share[buf], lane, wv, carry, s);
            const bool plain = __all(t.fl == 0 && t.n == K);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!plain) {
                    if (k >= t.n) continue;
                    const int f = t.flag(k);
                    if (f & REC_START) {
#pragma unroll
                        for (int v = 0; v < VEC; ++v) s[v] = a.h0 ? (Acc)widen(a.h0[a.ep[r0 + k] * a.ldh0 + cb + v]) : Acc(0);
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
                if (mine) {
                    __builtin_memcpy(a.h + (r0 + k) * a.sh + cb, &o, sizeof(o));
                    if (a.last && !plain && (t.flag(k) & REC_END)) __builtin_memcpy(a.last + a.ep[r0 + k] * a.D + cb, &o, sizeof(o));
                }
            }
        }
        t = next;
    }
    if constexpr (AGG) {
        if (mine && wv == 0 && lane < C)
            for (int v = 0; v < VEC; ++v) {
                a.agg[(int64_t)p * 2 * a.D + cb + v] = whole.A[v];
                a.agg[((int64_t)p * 2 + 1) * a.D + cb + v] = whole.B[v];
            }
    }
}

template <typename T, int C, int VEC, int GK, bool AGG>
__global__ __launch_bounds__(REC_THREADS) void rec_backward_kernel(RecWalk<T> a) {
    using Acc = typename SeqType<T>::Acc;
    constexpr int K = REC_K<T>, TILE = REC_TILE<C, T>;
    __shared__ RecShare<Acc, C, VEC> share_b[2], share_f[2];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane % C;
    const int64_t c0 = ((int64_t)blockIdx.x * C + c) * VEC;
    const bool mine = c0 < a.D;
    const int64_t cb = c0 < a.D - VEC ? c0 : a.D - VEC;
    if (!AGG && (int)blockIdx.y >= a.P) {                  // an empty episode hands its dlast through
        const int64_t step = (int64_t)(gridDim.y - a.P) * REC_WAVES * (64 / C);
        for (int64_t e = (((int64_t)blockIdx.y - a.P) * REC_WAVES + wv) * (64 / C) + lane / C; e < a.E; e += step)
            if (rec_ep_begin(a.ep_off, e, a.reverse, a.N) >= rec_ep_end(a.ep_off, e, a.reverse, a.N) && mine)
                for (int v = 0; v < VEC; ++v) a.dh0[e * a.D + cb + v] = a.dlast ? a.dlast[e * a.D + cb + v] : narrow<T>(0.0f);
        return;
    }
    const int p = blockIdx.y;
    const int64_t row0 = a.part[p];
    int64_t row1 = a.part[p + 1];
    if (row0 >= row1) return;
    Acc carry[VEC];
    RecMap<Acc, VEC> whole;
    if constexpr (AGG) {
        if (row0 == 0 || (a.flag[row0 - 1] & (REC_END | REC_OUT))) return;          // no episode comes in from before this part
        const int64_t e = rec_ep_end(a.ep_off, a.ep[row0 - 1], a.reverse, a.N);
        row1 = e < row1 && e > row0 ? e : row1;
        whole.one();
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) carry[v] = 0;
        if (row1 < a.N && !(a.flag[row1 - 1] & (REC_END | REC_OUT))) {
            const int64_t e = rec_ep_end(a.ep_off, a.ep[row1 - 1], a.reverse, a.N);       // one behind its last step
            int q = p + 1;
            while (q < a.P - 1 && a.part[q + 1] < e) ++q;
            for (bool first = true; q > p; --q, first = false) {
                if (a.part[q] >= a.part[q + 1]) continue;
                const Acc* m = a.agg + (int64_t)q * 2 * a.D + cb;
#pragma unroll
                for (int v = 0; v < VEC; ++v) carry[v] = first ? m[a.D + v] : fma(m[v], carry[v], m[a.D + v]);
            }
        }
    }
    const int64_t seg = (int64_t)(wv * (64 / C) + lane / C) * K;
    int64_t tiles = (row1 - row0 + TILE - 1) / TILE;
    int64_t base = row0 + (tiles - 1) * TILE, slot = row0 / TILE + p + tiles - 1;
    RecTile<T, C, VEC, GK, true> t, next;
    t.load(a, base + seg, row1, cb, !AGG);
    int buf = 0;
    for (; base >= row0; base -= TILE, buf ^= 1, --slot) {
        if (base > row0) next.load(a, base - TILE + seg, row1, cb, !AGG);
        const int64_t r0 = base + seg;
        RecMap<Acc, VEC> mb, mf;
        rec_map_backward(a, t, r0, cb, mb);
        rec_scan_wave<Acc, C, VEC, -1>(mb, share_b[buf], lane, wv);
        Acc state[VEC];
        if constexpr (!AGG) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) state[v] = a.state[slot * a.D + cb + v];
            rec_map_forward(a, t, r0, cb, mf);
            rec_scan_wave<Acc, C, VEC, 1>(mf, share_f[buf], lane, wv);
        }
        __syncthreads();
        if constexpr (AGG) {
#pragma unroll
            for (int w = REC_WAVES - 1; w >= 0; --w) {
                RecMap<Acc, VEC> f = whole;
                whole.cut = share_b[buf].cut[w] != 0;
#pragma unroll
                for (int v = 0; v < VEC; ++v) { whole.A[v] = share_b[buf].A[w][c * VEC + v]; whole.B[v] = share_b[buf].B[w][c * VEC + v]; }
                whole.after(f);
            }
        } else {
            Acc s[VEC], back[VEC], prev[K][VEC];
            rec_carry<Acc, C, VEC, -1>(mb, share_b[buf], lane, wv, carry, back);
            rec_carry<Acc, C, VEC, 1>(mf, share_f[buf], lane, wv, state, s);
#pragma unroll
            for (int k = 0; k < K; ++k) {                  // the states before each step once more, in 32 bits
                if (k < t.n && (t.flag(k) & REC_START)) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) s[v] = a.h0 ? (Acc)widen(a.h0[a.ep[r0 + k] * a.ldh0 + cb + v]) : Acc(0);
                }
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    prev[k][v] = s[v];
                    s[v] = fma(t.gate(a, k, v), s[v], (Acc)widen(t.x[k].v[v]));
                }
            }
            Acc sum[K];
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                sum[k] = 0;
                if (k >= t.n) continue;
                const int f = t.flag(k);
                if (f & REC_END) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) back[v] = a.dlast ? (Acc)widen(a.dlast[a.ep[r0 + k] * a.D + cb + v]) : Acc(0);
                }
                RecRaw<T, VEC> ox, og;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const Acc d = widen(t.dh[k].v[v]) + back[v], term = d * prev[k][v];
                    ox.v[v] = narrow<T>(d);
                    og.v[v] = narrow<T>(term);
                    if (GK == 1 && cb + v >= c0 && !(f & REC_OUT)) sum[k] += term;   // a channel counts in one lane only
                    back[v] = t.gate(a, k, v) * d;
                }
                if (f & REC_OUT) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) { ox.v[v] = og.v[v] = narrow<T>(0.0f); back[v] = 0; }
                }
                if (mine) {
                    if (a.dx) __builtin_memcpy(a.dx + (r0 + k) * a.sh + cb, &ox, sizeof(ox));
                    if (GK == 2 && a.dg) __builtin_memcpy(a.dg + (r0 + k) * a.sh + cb, &og, sizeof(og));
                    if (a.dh0 && (f & REC_START)) {
                        RecRaw<T, VEC> o0;
#pragma unroll
                        for (int v = 0; v < VEC; ++v) o0.v[v] = narrow<T>(back[v]);
                        __builtin_memcpy(a.dh0 + a.ep[r0 + k] * a.D + cb, &o0, sizeof(o0));
                    }
                }
            }
            if constexpr (GK == 1) {
                if (a.dg) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        Acc v = mine ? sum[k] : Acc(0);
#pragma unroll
                        for (int o = 1; o < C; o <<= 1) v += __shfl_xor(v, o);
                        if (c == 0 && k < t.n) {
                            if (a.dgp) a.dgp[(int64_t)blockIdx.x * a.N + r0 + k] = v;
                            else a.dg[(r0 + k) * (a.reverse ? -1 : 1)] = narrow<T>(v);
                        }
                    }
                }
            }
        }
        t = next;
    }
    if constexpr (AGG) {
        if (mine && wv == 0 && lane < C)
            for (int v = 0; v < VEC; ++v) {
                a.agg[(int64_t)p * 2 * a.D + cb + v] = whole.A[v];
                a.agg[((int64_t)p * 2 + 1) * a.D + cb + v] = whole.B[v];
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

// workgroups that look for empty episodes, beside those of the parts
inline unsigned rec_empty_blocks(bool wanted, int64_t E) { return wanted ? (unsigned)((E + 1023) / 1024 < 1024 ? (E + 1023) / 1024 : 1024) : 0; }

struct RecPlan {
    int P, blocks, tile;
    int64_t slots;
    int64_t flag, ep, part, plan_bytes;                    // the walk: in the states where there are any, else in the workspace
    int64_t state, states_bytes;
    int64_t agg, dgp, ws_plan, ws_bytes;
};
RecPlan rec_plan(int64_t N, int64_t D, int type, int gate_kind);

template <typename T> void rec_launch_forward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st);
template <typename T> void rec_launch_backward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st);

}  // namespace dcarl
