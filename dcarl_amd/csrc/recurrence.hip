// The recurrence along episodes: the walk's flags, the plan of a call, the launches of the forward pass (kernels: recurrence_impl.h).
#include <type_traits>
#include "recurrence_impl.h"

namespace dcarl {

// thread r < N: flags and episode of step r of the walk; threads N .. N + P: where part p begins
__global__ __launch_bounds__(256) void rec_walk_kernel(const int64_t* off, int64_t E, int64_t N, int reverse, int P, int64_t R, uint8_t* flag,
                                                       int32_t* ep, int64_t* part) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i > N + P) return;
    const int64_t p = i - N;
    if (p == 0 || p == P) { part[p] = p ? N : 0; return; }
    const int64_t r = p > 0 ? p * R : i;
    if (r >= N) { part[p] = N; return; }
    const int64_t t = reverse ? N - 1 - r : r;
    int64_t lo = 0, hi = E + 1;                            // the first offset above t
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid] <= t) lo = mid + 1; else hi = mid;
    }
    const bool out = lo == 0 || lo > E;
    const int64_t e = out ? 0 : lo - 1;
    if (p > 0) {
        int64_t at = r;
        if (!out) {                                        // the nearest start within a quarter of a part
            const int64_t s0 = rec_ep_begin(off, e, reverse, N), s1 = rec_ep_end(off, e, reverse, N);
            const int64_t b = r - s0, f = s1 - r;
            if (b <= f && b <= R / 4) at = s0;
            else if (f < b && f <= R / 4) at = s1;
        }
        part[p] = at;
    } else {
        int f = REC_OUT;
        if (!out) {
            const bool first = t == off[e], last = t == off[e + 1] - 1;
            f = ((reverse ? last : first) ? REC_START : 0) | ((reverse ? first : last) ? REC_END : 0);
        }
        flag[r] = (uint8_t)f;
        ep[r] = (int32_t)e;
    }
}

template <typename T> __global__ __launch_bounds__(256) void rec_share_kernel(const typename SeqType<T>::Acc* dgp, int blocks, int64_t N, int step, T* dg) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= N) return;
    typename SeqType<T>::Acc s = 0;
    for (int b = 0; b < blocks; ++b) s += dgp[b * N + r];
    dg[r * step] = narrow<T>(s);
}

static int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }

RecPlan rec_plan(int64_t N, int64_t D, int type, int gate_kind) {
    RecPlan p{};
    const int64_t acc = type == DCARL_F64 ? 8 : 4;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        rec_with_shape<T>(D, [&](auto C, auto V) {
            p.tile = REC_TILE<C(), T>;
            p.blocks = (int)((D + C() * V() - 1) / (C() * V()));
        });
    });
    // as many parts as give every CU a few workgroups, none under two tiles
    int64_t want = (1024 + p.blocks - 1) / p.blocks, most = N / (2 * p.tile);
    want = want < most ? want : most;
    p.P = (int)(want < 1 ? 1 : want > REC_MAX_PARTS ? REC_MAX_PARTS : want);
    p.slots = N / p.tile + p.P + 1;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at += up16(bytes); return here; };
    p.flag = take(N + 8); p.ep = take(4 * N); p.part = take(8 * (p.P + 1));
    p.plan_bytes = at;
    p.state = take(p.slots * D * acc);
    p.states_bytes = at;
    at = 0;
    p.ws_plan = take(p.plan_bytes);
    p.agg = take(p.P > 1 ? 2 * p.P * D * acc : 0);
    p.dgp = take(gate_kind == 1 && p.blocks > 1 ? p.blocks * N * acc : 0);
    p.ws_bytes = at;
    return p;
}
int64_t recurrence_workspace_bytes(int64_t N, int64_t D, int64_t, int type, int gate_kind) { return D ? rec_plan(N, D, type, gate_kind).ws_bytes : 0; }
int64_t recurrence_states_bytes(int64_t N, int64_t D, int64_t, int type, int gate_kind) { return D ? rec_plan(N, D, type, gate_kind).states_bytes : 0; }

template <typename T> static RecWalk<T> rec_walk(const dcarl_recurrence_t& r, const RecPlan& p, char* plan, char* ws) {
    using Acc = typename SeqType<T>::Acc;
    RecWalk<T> a{};
    a.N = r.N; a.D = r.D; a.E = r.E; a.ep_off = r.ep_off; a.reverse = r.reverse; a.P = p.P;
    const int64_t top = r.reverse ? r.N - 1 : 0, dir = r.reverse ? -1 : 1;
    a.x = static_cast<const T*>(r.x) + top * r.ldx; a.sx = dir * r.ldx;
    a.g = r.gate_kind ? static_cast<const T*>(r.gate) + top * r.ldg : nullptr; a.sg = dir * r.ldg;
    a.h0 = static_cast<const T*>(r.h0); a.ldh0 = r.ldh0;
    a.gval = (Acc)r.gate_value;
    a.flag = reinterpret_cast<uint8_t*>(plan + p.flag);
    a.ep = reinterpret_cast<int32_t*>(plan + p.ep);
    a.part = reinterpret_cast<int64_t*>(plan + p.part);
    a.agg = reinterpret_cast<Acc*>(ws + p.agg);
    a.sh = dir * r.D;
    return a;
}

template <typename T> void rec_launch_forward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st) {
    rec_with_shape<T>(a.D, [&](auto C, auto V) {
        auto go = [&](auto GK) {
            if (p.P > 1)
                hipLaunchKernelGGL((rec_forward_kernel<T, C(), V(), GK(), true>), dim3(p.blocks, p.P - 1), dim3(REC_THREADS), 0, st, a);
            const unsigned empty = rec_empty_blocks(a.last, a.E);
            hipLaunchKernelGGL((rec_forward_kernel<T, C(), V(), GK(), false>), dim3(p.blocks, p.P + empty), dim3(REC_THREADS), 0, st, a);
        };
        if (gate_kind == 2) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 1>{});
    });
}

static void rec_launch_walk(const dcarl_recurrence_t& r, const RecPlan& p, char* plan, hipStream_t st) {
    const int64_t R = (r.N + p.P - 1) / p.P;
    hipLaunchKernelGGL(rec_walk_kernel, dim3((unsigned)((r.N + p.P) / 256 + 1)), dim3(256), 0, st, r.ep_off, r.E, r.N, r.reverse, p.P, R,
                       reinterpret_cast<uint8_t*>(plan + p.flag), reinterpret_cast<int32_t*>(plan + p.ep), reinterpret_cast<int64_t*>(plan + p.part));
}

void launch_recurrence_forward(const dcarl_recurrence_t& r, void* states, void* workspace, void* h, void* last, hipStream_t st) {
    const RecPlan p = rec_plan(r.N, r.D, r.type, r.gate_kind);
    char* ws = static_cast<char*>(workspace);
    char* plan = states ? static_cast<char*>(states) : ws + p.ws_plan;
    rec_launch_walk(r, p, plan, st);
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        RecWalk<T> a = rec_walk<T>(r, p, plan, ws);
        a.h = static_cast<T*>(h) + (r.reverse ? (r.N - 1) * r.D : 0);
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
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        RecWalk<T> a = rec_walk<T>(r, p, plan, ws);
        a.state = reinterpret_cast<Acc*>(plan + p.state);
        const int64_t top = r.reverse ? r.N - 1 : 0;
        a.dh = static_cast<const T*>(dh) + top * lddh; a.sdh = (r.reverse ? -1 : 1) * lddh;
        a.dlast = static_cast<const T*>(dlast);
        a.dx = dx ? static_cast<T*>(dx) + top * r.D : nullptr;
        a.dg = dgate ? static_cast<T*>(dgate) + top * (r.gate_kind == 2 ? r.D : 1) : nullptr;
        a.dh0 = static_cast<T*>(dh0);
        a.dgp = r.gate_kind == 1 && p.blocks > 1 ? reinterpret_cast<Acc*>(ws + p.dgp) : nullptr;
        rec_launch_backward<T>(a, r.gate_kind, p, st);
        if (a.dgp && a.dg)
            hipLaunchKernelGGL((rec_share_kernel<T>), dim3((unsigned)((r.N + 255) / 256)), dim3(256), 0, st, a.dgp, p.blocks, r.N, r.reverse ? -1 : 1, a.dg);
    });
}

}  // namespace dcarl
