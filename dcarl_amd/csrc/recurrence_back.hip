// The recurrence along episodes: the launches of the backward pass (kernels: recurrence_impl.h).
#include <type_traits>
#include "recurrence_impl.h"

namespace dcarl {

template <typename T> void rec_launch_backward(const RecWalk<T>& a, int gate_kind, const RecPlan& p, hipStream_t st) {
    rec_with_shape<T>(a.D, [&](auto C, auto V) {
        auto go = [&](auto GK) {
            const dim3 grid((unsigned)(p.tiles * p.blocks + rec_empty_blocks(a.dh0, a.E)));
            if (grid.x) hipLaunchKernelGGL((rec_backward_kernel<T, C(), V(), GK()>), grid, dim3(REC_THREADS), 0, st, a);
        };
        if (gate_kind == 2) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 1>{});
    });
}

int recurrence_status_backward() { return rec_take(); }

template void rec_launch_backward<double>(const RecWalk<double>&, int, const RecPlan&, hipStream_t);
template void rec_launch_backward<float>(const RecWalk<float>&, int, const RecPlan&, hipStream_t);
template void rec_launch_backward<bf16>(const RecWalk<bf16>&, int, const RecPlan&, hipStream_t);
template void rec_launch_backward<f16>(const RecWalk<f16>&, int, const RecPlan&, hipStream_t);

}  // namespace dcarl
