// The experts' choice of route.cu for the layer calls of moe.cu.
#pragma once
#include "common.cuh"
#include "../../include/berth_b200.h"

namespace berth {

// Throws on values out of range (r is not null).
void check_routing(const berth_moe_routing* r, int n_experts, int top_k);
// idx / w [T][k] from logits [T] of row stride ld; r checked.  Returns the name of the kernel that runs.
std::string route_tokens(const void* logits, bool f32, long long ld, const berth_moe_routing& r, int32_t* idx, float* w, int T, int E, int k,
                         cudaStream_t st);

}  // namespace berth
