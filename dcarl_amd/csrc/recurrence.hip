// The recurrence along episodes: the walk's flags, the plan of a call, the launches of the forward pass (kernels: recurrence_impl.h).
#include <atomic>
#include <type_traits>
#include "recurrence_impl.h"

namespace dcarl {

// flags and episode of every step of the walk, `finds` of them per thread; where the episodes that cross a tile's borders begin and end.  tile: 1 << tile_bits steps
__global__ __launch_bounds__(256) void rec_walk_kernel(const int64_t* off, int64_t E, int64_t N, int reverse, int tile_bits, int finds, int64_t tiles, uint8_t* flag,
                                                       int32_t* ep, int32_t* from, int32_t* till, uint32_t* ticket, int64_t blocks, uint4* clear, int64_t clear16) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    for (int64_t k = i; k < blocks; k += all) ticket[k * REC_TICKET] = 0;
    for (int64_t k = i; k < clear16; k += all) clear[k] = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (!off) return;
    RecFind find;
    for (int64_t r = i * finds; r < (i + 1) * finds && r < N; ++r) {
        const int f = find.at(off, E, N, reverse, r);
        const bool out = f & REC_OUT;
        flag[r] = (uint8_t)f;
        if (ep) ep[r] = (int32_t)find.e;
        // (held inside the walk whatever the offsets say: a tile waits for tiles between itself and these)
        const int64_t at = r >> tile_bits, lr = r - (at << tile_bits);
        if (lr == 0) {
            const int64_t b = out || (f & REC_START) || at == 0 ? -1 : rec_ep_begin(off, find.e, reverse, N) >> tile_bits;
            from[at] = (int32_t)(b >= at ? at - 1 : b);
        }
        if (lr == (1 << tile_bits) - 1 || r == N - 1) {
            const int64_t z = out || (f & REC_END) || at + 1 == tiles ? -1 : (rec_ep_end(off, find.e, reverse, N) - 1) >> tile_bits;
            till[at] = (int32_t)(z >= 0 && z <= at ? at + 1 : z);
        }
    }
}

// One step of every live episode: a thread takes VEC channels of an episode from its first step to its last, REC_DEEP steps on the way at a time.
// Nothing to find and to join, and a fraction of the tiles' code, whose fetch is most of what a tile by itself costs.  Bound by two waits for memory.
constexpr int REC_DEEP = 8, REC_LIVE_STEPS = 128, REC_LIVE = 1024;
template <typename T, int VEC, int GK> __global__ __launch_bounds__(REC_THREADS) void rec_step_kernel(RecWalk<T> a, uint32_t vecs) {
    using Acc = typename SeqType<T>::Acc;
    const uint32_t i = blockIdx.x * (uint32_t)REC_THREADS + threadIdx.x, e = i / vecs;
    const int64_t c0 = (int64_t)(i - e * vecs) * VEC;
    const uint32_t cb = (uint32_t)(c0 < a.D - VEC ? c0 : a.D - VEC);       // the last one moves back to a whole vector: the same values
    RecRaw<T, VEC> o;
    if (e >= a.E) {                                        // what lies outside the episodes
        if (e > a.E) return;
        const int64_t front = rec_ep_begin(a.ep_off, 0, 0, a.N), behind = rec_ep_end(a.ep_off, a.E - 1, 0, a.N);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o.v[v] = narrow<T>(0.0f);
        for (int64_t t = 0; t < front; ++t) __builtin_memcpy(a.h + t * a.D + cb, &o, sizeof(o));
        for (int64_t t = behind; t < a.N; ++t) __builtin_memcpy(a.h + t * a.D + cb, &o, sizeof(o));
        if (a.state)
            for (int v = 0; v < VEC; ++v) a.state[cb + v] = 0;                                   // nothing comes into the one tile
        return;
    }
    const int from = (int)rec_ep_begin(a.ep_off, e, 0, a.N), n = (int)rec_ep_end(a.ep_off, e, 0, a.N) - from;
    auto step = [&](int k) { return (uint32_t)(from + (a.reverse ? n - 1 - k : k)); };
    Acc s[VEC];
    if (a.h0) __builtin_memcpy(&o, a.h0 + (int64_t)e * a.ldh0 + cb, sizeof(o));
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        o.v[v] = a.h0 ? o.v[v] : narrow<T>(0.0f);
        s[v] = widen(o.v[v]);
    }
    const T* gate = a.g ? a.g : a.x;                       // (a gate that is a number: something to load)
    const uint32_t gate_step = a.g ? a.ldg : 0, gate_at = GK == 2 ? cb : 0;
    auto some = [&](int k, auto M) {                   // M steps from k on, as many of them as there are
        RecRaw<T, VEC> x[M()];
        RecRaw<T, GK == 2 ? VEC : 1> g[M()];
#pragma unroll
        for (int j = 0; j < M(); ++j) {
            const uint32_t t = step(k + j < n ? k + j : n - 1);
            x[j] = rec_load<T, VEC>(a.x, t * a.ldx + cb);
            g[j] = rec_load<T, GK == 2 ? VEC : 1>(gate, t * gate_step + gate_at);
        }
#pragma unroll
        for (int j = 0; j < M(); ++j)
            if (k + j < n) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    s[v] = fma(GK == 2 || a.g ? (Acc)widen(g[j].v[GK == 2 ? v : 0]) : a.gval, s[v], (Acc)widen(x[j].v[v]));
                    o.v[v] = narrow<T>(s[v]);
                }
                rec_store(a.h, step(k + j) * (uint32_t)a.D + cb, o, false);
            }
    };
    if (n > 0) some(0, std::integral_constant<int, 1>{});
    for (int k = 1; k < n; k += REC_DEEP) some(k, std::integral_constant<int, REC_DEEP>{});
    if (a.last) __builtin_memcpy(a.last + (int64_t)e * a.D + cb, &o, sizeof(o));
}

template <typename T> __global__ __launch_bounds__(256) void rec_share_kernel(const typename SeqType<T>::Acc* dgp, int blocks, int64_t N, int reverse, T* dg) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= N) return;
    typename SeqType<T>::Acc s = 0;
    for (int b = 0; b < blocks; ++b) s += dgp[b * N + r];
    dg[reverse ? N - 1 - r : r] = narrow<T>(s);
}

static std::atomic<int> rec_polls{REC_POLLS};              // (a test hook lowers it)
void recurrence_polls(int polls) { rec_polls = polls < 0 || polls > REC_POLLS ? REC_POLLS : polls; }
int recurrence_status(hipStream_t st) {
    if (hipStreamSynchronize(st) != hipSuccess) return -1;
    const int f = rec_take(), b = recurrence_status_backward();
    return f < 0 || b < 0 ? -1 : f | b;
}

static int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }

RecPlan rec_plan(int64_t N, int64_t D, int type, int gate_kind) {
    RecPlan p{};
    const int64_t acc = type == DCARL_F64 ? 8 : 4;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        rec_with_shape<T>(D, [&](auto C, auto V) {
            p.tile = REC_TILE<C(), T>;
            p.blocks = (D + C() * V() - 1) / (C() * V());
            p.wide = p.blocks * C() * V();
        });
    });
    p.tiles = (N + p.tile - 1) / p.tile;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at += up16(bytes); return here; };
    p.flag = take(N + 16); p.ep = take(4 * N); p.from = take(4 * p.tiles); p.till = take(4 * p.tiles);
    p.plan_bytes = at;
    p.state = take(p.tiles * D * acc);
    p.states_bytes = at;
    at = 0;
    p.map = take(p.tiles > 1 ? 2 * p.tiles * p.wide * acc : 0);
    p.group = take(p.tiles > 1 ? 2 * (p.tiles / REC_GROUP + 1) * p.wide * acc : 0);
    p.through = take(p.tiles > 1 ? (p.tiles / REC_GROUP + 1) * p.wide * acc : 0);
    p.clear_bytes = at;
    p.ticket = take(p.tiles > 1 ? 4 * REC_TICKET * p.blocks : 0);
    p.ws_plan = take(p.tiles > 1 ? p.plan_bytes : 0);
    p.dgp = take(gate_kind == 1 && p.blocks > 1 ? p.blocks * N * acc : 0);
    p.ws_bytes = at;
    return p;
}
// the largest row distance: a tile's rows are addressed by 32-bit offsets
int64_t recurrence_max_ld(int64_t D, int type) {
    return ((int64_t)1 << 31) / rec_plan(1, D, type, 2).tile / (type == DCARL_F64 ? 8 : type == DCARL_F32 ? 4 : 2);
}
// workgroups of a call's largest launch
int64_t recurrence_workgroups(int64_t N, int64_t D, int64_t E, int type) {
    const RecPlan p = rec_plan(N, D, type, 2);
    return p.tiles * p.blocks + rec_empty_blocks(true, E);
}
int64_t recurrence_workspace_bytes(int64_t N, int64_t D, int64_t, int type, int gate_kind) { return D ? rec_plan(N, D, type, gate_kind).ws_bytes : 0; }
int64_t recurrence_states_bytes(int64_t N, int64_t D, int64_t, int type, int gate_kind) { return D ? rec_plan(N, D, type, gate_kind).states_bytes : 0; }

template <typename T> static RecWalk<T> rec_walk(const dcarl_recurrence_t& r, const RecPlan& p, char* plan, char* ws) {
    using Acc = typename SeqType<T>::Acc;
    RecWalk<T> a{};
    a.N = r.N; a.D = r.D; a.E = r.E; a.ep_off = r.ep_off; a.reverse = r.reverse; a.polls = rec_polls; a.past = r.D * sizeof(T) % 128 == 0; a.tiles = p.tiles; a.blocks = p.blocks;
    a.x = static_cast<const T*>(r.x); a.ldx = (uint32_t)r.ldx;
    a.g = r.gate_kind ? static_cast<const T*>(r.gate) : nullptr; a.ldg = (uint32_t)r.ldg;
    a.h0 = r.E ? static_cast<const T*>(r.h0) : nullptr; a.ldh0 = r.ldh0;       // (without episodes it has no row, and row 0 is read for steps that start none)
    a.gval = (Acc)r.gate_value;
    if (p.tiles <= 1) return a;                            // finds its flags itself, waits for nothing
    a.flag = reinterpret_cast<uint8_t*>(plan + p.flag);
    a.ep = reinterpret_cast<int32_t*>(plan + p.ep);
    a.ticket = reinterpret_cast<uint32_t*>(ws + p.ticket);
    a.map = reinterpret_cast<Acc*>(ws + p.map);
    a.group = reinterpret_cast<Acc*>(ws + p.group);
    a.through = reinterpret_cast<Acc*>(ws + p.through);
    a.from = reinterpret_cast<int32_t*>(plan + p.from);
    a.till = reinterpret_cast<int32_t*>(plan + p.till);
    return a;
}

template <typename T> void rec_launch_forward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st) {
    // A few episodes of about a step each: by episode.  In a graph, 48 steps of 48 episodes of 768 bf16 channels: 2.0 us (as a tile 8.7); 128 of 128, 2048 channels:
    // 2.0 (8.9); two steps each, 96 of 48: 2.4 (8.4).  At worst all but one of them are empty, and the threads of that one walk all: 64 steps 9 (9), 128 16 (9).
    if (p.tiles == 1 && a.N <= REC_LIVE_STEPS && a.N <= 2 * a.E && a.E <= REC_LIVE) {
        auto go = [&](auto V) {
            const int64_t vecs = (a.D + V() - 1) / V();
            const dim3 grid((unsigned)(((a.E + 1) * vecs + REC_THREADS - 1) / REC_THREADS));
            if (gate_kind == 2) hipLaunchKernelGGL((rec_step_kernel<T, V(), 2>), grid, dim3(REC_THREADS), 0, st, a, (uint32_t)vecs);
            else hipLaunchKernelGGL((rec_step_kernel<T, V(), 1>), grid, dim3(REC_THREADS), 0, st, a, (uint32_t)vecs);
        };
        if (a.D >= REC_VEC<T>) go(std::integral_constant<int, REC_VEC<T>>{});
        else go(std::integral_constant<int, 1>{});
        return;
    }
    rec_with_shape<T>(a.D, [&](auto C, auto V) {
        auto go = [&](auto GK) {
            const dim3 grid((unsigned)(p.tiles * p.blocks + rec_empty_blocks(a.last, a.E)));
            if (grid.x) hipLaunchKernelGGL((rec_forward_kernel<T, C(), V(), GK()>), grid, dim3(REC_THREADS), 0, st, a);
        };
        if (gate_kind == 2) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 1>{});
    });
}

// the walk (off given) and what the launch behind it needs cleared
static void rec_launch_walk(const dcarl_recurrence_t& r, const RecPlan& p, const int64_t* off, bool episodes, char* plan, char* ws, hipStream_t st) {
    // one step per thread ends soonest (400000 steps: 4.6 us, with four 7.9); four where there are more steps than the GPU holds threads (4e6: 52 -> 43 us)
    const int finds = r.N >= (1 << 20) ? 4 : 1;
    hipLaunchKernelGGL(rec_walk_kernel, dim3((unsigned)(r.N / (256 * finds) + 1)), dim3(256), 0, st, off, r.E, r.N, r.reverse, __builtin_ctz((unsigned)p.tile), finds, p.tiles,
                       reinterpret_cast<uint8_t*>(plan + p.flag), episodes ? reinterpret_cast<int32_t*>(plan + p.ep) : nullptr,
                       reinterpret_cast<int32_t*>(plan + p.from), reinterpret_cast<int32_t*>(plan + p.till), reinterpret_cast<uint32_t*>(ws + p.ticket),
                       p.tiles > 1 ? p.blocks : 0, reinterpret_cast<uint4*>(ws), p.clear_bytes / 16);
}

void launch_recurrence_forward(const dcarl_recurrence_t& r, void* states, void* workspace, void* h, void* last, hipStream_t st) {
    const RecPlan p = rec_plan(r.N, r.D, r.type, r.gate_kind);
    char* ws = static_cast<char*>(workspace);
    char* plan = states ? static_cast<char*>(states) : ws + p.ws_plan;
    if (p.tiles > 1) rec_launch_walk(r, p, r.ep_off, r.h0 || last || states, plan, ws, st);     // (a backward pass may ask for dh0 or bring a dlast)
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        RecWalk<T> a = rec_walk<T>(r, p, plan, ws);
        a.h = static_cast<T*>(h);
        a.last = static_cast<T*>(last);
        if (states) a.state = reinterpret_cast<typename SeqType<T>::Acc*>(plan + p.state);
        rec_launch_forward<T>(a, r.gate_kind, p, st);
    });
}

void launch_recurrence_backward(const dcarl_recurrence_t& r, const void* states, void* workspace, const void* dh, int64_t lddh, const void* dlast,
                                void* dx, void* dgate, void* dh0, hipStream_t st) {
    const RecPlan p = rec_plan(r.N, r.D, r.type, r.gate_kind);
    char* ws = static_cast<char*>(workspace);
    char* plan = static_cast<char*>(const_cast<void*>(states));
    if (p.tiles > 1) rec_launch_walk(r, p, nullptr, false, plan, ws, st);
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        RecWalk<T> a = rec_walk<T>(r, p, plan, ws);
        a.state = reinterpret_cast<Acc*>(plan + p.state);
        a.dh = static_cast<const T*>(dh); a.lddh = (uint32_t)lddh;
        a.dlast = r.E ? static_cast<const T*>(dlast) : nullptr;
        a.dx = static_cast<T*>(dx);
        a.dg = static_cast<T*>(dgate);
        a.dh0 = r.E ? static_cast<T*>(dh0) : nullptr;
        a.dgp = r.gate_kind == 1 && p.blocks > 1 ? reinterpret_cast<Acc*>(ws + p.dgp) : nullptr;
        rec_launch_backward<T>(a, r.gate_kind, p, st);
        if (a.dgp && a.dg)
            hipLaunchKernelGGL((rec_share_kernel<T>), dim3((unsigned)((r.N + 255) / 256)), dim3(256), 0, st, a.dgp, (int)p.blocks, r.N, r.reverse, a.dg);
    });
}

}  // namespace dcarl
