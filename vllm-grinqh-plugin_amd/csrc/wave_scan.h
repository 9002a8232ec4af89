// Sums over the lanes of a wave by lane permutes (no LDS round trips).
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

namespace grinqh {

// Inclusive sum over the lanes of a wave (row shifts, then the rows' totals).
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  auto step = [&](auto ctrl, auto rows) {
    const int x = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                              decltype(rows)::value, 0xf, false);
    v += __builtin_bit_cast(T, x);
  };
  using I = std::integral_constant<int, 0xf>;
  step(std::integral_constant<int, 0x111>{}, I{});
  step(std::integral_constant<int, 0x112>{}, I{});
  step(std::integral_constant<int, 0x114>{}, I{});
  step(std::integral_constant<int, 0x118>{}, I{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return v;
}

// op over all lanes, in all of them (scalar), for an op with op(x, x) == x.
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T v, F&& op) {
  auto step = [&](auto ctrl, auto rows) {
    const int own = __builtin_bit_cast(int, v);
    v = op(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(own, own, decltype(ctrl)::value, decltype(rows)::value,
                                                               0xf, false)));
  };
  using I = std::integral_constant<int, 0xf>;
  step(std::integral_constant<int, 0x111>{}, I{});
  step(std::integral_constant<int, 0x112>{}, I{});
  step(std::integral_constant<int, 0x114>{}, I{});
  step(std::integral_constant<int, 0x118>{}, I{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Sum of all lanes, in all of them (scalar).
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

}  // namespace grinqh
