// Routing of bf16 logits, see d2d_route.cuh.
#include "d2d_route.cuh"

namespace d2d {

int launch_route_bf16(const RouteCall& c, int sms, cudaStream_t s) {
  const int size = c.E / c.groups;
  const RouteArgs a = {c.logits, c.bias, c.experts, c.weights, c.mask_bits, c.dense, c.N, c.E, c.k, c.groups,
                       c.top_groups, c.softmax, c.renormalise, c.scale, 0,
                       (reinterpret_cast<uintptr_t>(c.bias) & 15) == 0, ((1u << 22) + size - 1) / size};
  return route_t<bf16>(a, sms, s);
}

int launch_route_backward_bf16(const RouteCall& c, const float* dweights, void* dlogits, int sms, cudaStream_t s) {
  const BackwardArgs a = {c.logits, c.experts, c.weights, dweights, dlogits, c.N, c.E, c.k, c.softmax, c.renormalise,
                          c.scale};
  return route_backward_t<bf16>(a, sms, s);
}

}  // namespace d2d
