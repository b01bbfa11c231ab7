// Gated linear recurrence along ragged episodes: h_t = g_t * h_{t-1} + x_t per channel, restarted from h0[e] (or 0) where episode e
// begins, and its gradients  d_t = dh_t + g_{t+1} d_{t+1},  dx = d,  dg_t = d_t h_{t-1},  dh0[e] = g_s d_s (s: the episode's first
// step).  `reverse` mirrors time: the host passes the last row's address and negative row strides, and the kernels read the
// offsets mirrored.
#include "seq_common.h"

namespace dcarl {

struct RecArgs {
    int64_t N, D, E;
    const int64_t* ep_off;
    const void *x, *gate, *h0;
    int64_t ldx, ldg, ldh0;
    double gate_value;
    int gate_kind, reverse;
};

// rows [b, e) of episode `ep`, clamped into [0, N) whatever the offsets hold; in walking order for `reverse`
__device__ __forceinline__ void rec_span(const RecArgs& a, int64_t ep, int64_t& b, int64_t& e) {
    b = a.ep_off[ep]; e = a.ep_off[ep + 1];
    b = b < 0 ? 0 : b > a.N ? a.N : b;
    e = e < b ? b : e > a.N ? a.N : e;
}

template <typename T>
__global__ __launch_bounds__(64) void rec_forward_kernel(RecArgs a, typename SeqType<T>::Acc* states, T* h, int64_t ldh, T* last) {
    using Acc = typename SeqType<T>::Acc;
    const int64_t d = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (d >= a.D) return;
    for (int64_t ep = blockIdx.y; ep < a.E; ep += gridDim.y) {
        int64_t b, e;
        rec_span(a, ep, b, e);
        Acc s = a.h0 ? widen(static_cast<const T*>(a.h0)[ep * a.ldh0 + d]) : Acc(0);
        for (int64_t i = 0; i < e - b; ++i) {
            const int64_t t = a.reverse ? e - 1 - i : b + i;
            const Acc g = a.gate_kind == 0 ? (Acc)a.gate_value
                          : widen(static_cast<const T*>(a.gate)[t * a.ldg + (a.gate_kind == 2 ? d : 0)]);
            if (states) states[t * a.D + d] = s;            // the state BEFORE step t
            s = g * s + widen(static_cast<const T*>(a.x)[t * a.ldx + d]);
            h[t * ldh + d] = narrow<T>(s);
        }
        if (last) last[ep * a.D + d] = narrow<T>(s);
    }
}

template <typename T>
__global__ __launch_bounds__(64) void rec_backward_kernel(RecArgs a, const typename SeqType<T>::Acc* states, const T* dh, int64_t lddh,
                                                          const T* dlast, T* dx, T* dgate, T* dh0, typename SeqType<T>::Acc* terms) {
    using Acc = typename SeqType<T>::Acc;
    const int64_t d = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (d >= a.D) return;
    for (int64_t ep = blockIdx.y; ep < a.E; ep += gridDim.y) {
        int64_t b, e;
        rec_span(a, ep, b, e);
        Acc c = dlast ? widen(dlast[ep * a.D + d]) : Acc(0);
        for (int64_t i = e - b - 1; i >= 0; --i) {
            const int64_t t = a.reverse ? e - 1 - i : b + i;
            const Acc g = a.gate_kind == 0 ? (Acc)a.gate_value
                          : widen(static_cast<const T*>(a.gate)[t * a.ldg + (a.gate_kind == 2 ? d : 0)]);
            const Acc dt = widen(dh[t * lddh + d]) + c;
            if (dx) dx[t * a.D + d] = narrow<T>(dt);
            const Acc term = dt * states[t * a.D + d];
            if (terms) terms[t * a.D + d] = term;
            else if (dgate) dgate[t * a.D + d] = narrow<T>(term);
            c = g * dt;
        }
        if (dh0) dh0[ep * a.D + d] = narrow<T>(c);
    }
}

// dgate[t] = sum over the channels of one step, for a gate that all channels share: one wavefront per step, a fixed butterfly
template <typename T>
__global__ __launch_bounds__(64) void rec_share_kernel(const typename SeqType<T>::Acc* terms, int64_t N, int64_t D, const int64_t* ep_off,
                                                       int64_t E, T* dgate) {
    using Acc = typename SeqType<T>::Acc;
    const int64_t n = E > 0 ? ep_off[E] : 0;
    for (int64_t t = blockIdx.x; t < N; t += gridDim.x) {
        Acc s = 0;
        if (t < n) for (int64_t d = threadIdx.x; d < D; d += 64) s += terms[t * D + d];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (threadIdx.x == 0) dgate[t] = narrow<T>(s);
    }
}

// rows behind the last episode: zeros in what the call makes
template <typename T>
__global__ __launch_bounds__(256) void rec_tail_kernel(const int64_t* ep_off, int64_t E, int64_t N, int64_t D, T* a, T* b, T* c) {
    int64_t n = E > 0 ? ep_off[E] : 0;
    n = n < 0 ? 0 : n;
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = n * D + (int64_t)blockIdx.x * 256 + threadIdx.x; i < N * D; i += step) {
        if (a) a[i] = narrow<T>(0.0f);
        if (b) b[i] = narrow<T>(0.0f);
        if (c) c[i] = narrow<T>(0.0f);
    }
}

static RecArgs rec_args(const dcarl_recurrence_t& r) {
    return RecArgs{r.N, r.D, r.E, r.ep_off, r.x, r.gate, r.h0, r.ldx, r.ldg, r.ldh0, r.gate_value, r.gate_kind, r.reverse};
}

int64_t recurrence_workspace_bytes(int64_t N, int64_t D, int64_t, int type, int gate_kind) {
    return gate_kind == 1 ? N * D * (type == DCARL_F64 ? 8 : 4) : 0;
}
int64_t recurrence_states_bytes(int64_t N, int64_t D, int64_t, int type, int) { return N * D * (type == DCARL_F64 ? 8 : 4); }

static dim3 rec_grid(const dcarl_recurrence_t& r) {
    return dim3((unsigned)((r.D + 63) / 64), (unsigned)(r.E < 65535 ? r.E : 65535));
}

void launch_recurrence_forward(const dcarl_recurrence_t& r, void* states, void*, void* h, void* last, hipStream_t st) {
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        if (r.N > 0)
            hipLaunchKernelGGL((rec_tail_kernel<T>), dim3(256), dim3(256), 0, st, r.ep_off, r.E, r.N, r.D, (T*)h, (T*)nullptr, (T*)nullptr);
        if (r.E > 0)
            hipLaunchKernelGGL((rec_forward_kernel<T>), rec_grid(r), dim3(64), 0, st, rec_args(r), (Acc*)states, (T*)h, r.D, (T*)last);
    });
}

void launch_recurrence_backward(const dcarl_recurrence_t& r, const void* states, void* ws, const void* dh, int64_t lddh, const void* dlast,
                                void* dx, void* dgate, void* dh0, hipStream_t st) {
    with_type(r.type, [&](auto t) {
        using T = decltype(t);
        using Acc = typename SeqType<T>::Acc;
        Acc* terms = r.gate_kind == 1 && dgate ? (Acc*)ws : nullptr;
        if (r.N > 0)
            hipLaunchKernelGGL((rec_tail_kernel<T>), dim3(256), dim3(256), 0, st, r.ep_off, r.E, r.N, r.D, (T*)dx,
                               r.gate_kind == 2 ? (T*)dgate : (T*)nullptr, (T*)nullptr);
        if (r.E > 0)
            hipLaunchKernelGGL((rec_backward_kernel<T>), rec_grid(r), dim3(64), 0, st, rec_args(r), (const Acc*)states, (const T*)dh, lddh,
                               (const T*)dlast, (T*)dx, r.gate_kind == 2 ? (T*)dgate : (T*)nullptr, (T*)dh0, terms);
        if (terms && r.N > 0)
            hipLaunchKernelGGL((rec_share_kernel<T>), dim3((unsigned)(r.N < 16384 ? r.N : 16384)), dim3(64), 0, st, terms, r.N, r.D, r.ep_off,
                               r.E, (T*)dgate);
    });
}

}  // namespace dcarl
