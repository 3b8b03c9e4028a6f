// Kernels' template arguments from values that a call brings.
#pragma once
#include <type_traits>

#include "values.cuh"

namespace b200 {

// f(element type) for one of the float types
template <class F>
auto with_float(int type, F f) {
    return type == B200_TYPE_F32 ? f(float{}) : type == B200_TYPE_BF16 ? f(bf16{}) : f(f16{});
}
template <class F>
void with_bool(bool b, F f) {
    if (b)
        f(std::true_type{});
    else
        f(std::false_type{});
}

}  // namespace b200
