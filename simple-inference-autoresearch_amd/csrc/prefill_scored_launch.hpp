// Launch of prefill_fwd with a score function at one head_dim.
#pragma once

#include "host_util.hpp"
#include "prefill_kernel.hpp"
#include "prefill_launch.hpp"

namespace sia {

template <int D, class T, int VAR, int MOD>
static int launch_scored_mod(PrefillLaunch& L) {
  ScoredPrefillArgs a;
  (PrefillArgs&)a = L.a;
  a.s = L.s;
  constexpr bool kSplit = PfCfg<D, VAR>::split;
  hipLaunchKernelGGL((prefill_fwd<D, T, kRopeNone, VAR, MOD>), dim3(L.a.nqblk * L.a.nunit * (kSplit ? L.a.nsplit : 1)),
                     dim3(PfCfg<D, VAR>::waves * 64), 0, L.stream, a);
  hipError_t e = hipGetLastError();
  if constexpr (kSplit) {
    if (e != hipSuccess) return fail(SIA_ERR_LAUNCH, "scored prefill launch: %s", hipGetErrorString(e));
    constexpr int RPB = 256 / (D / 4);
    hipLaunchKernelGGL((prefill_merge<D, T, kModMask>), dim3((unsigned)((L.a.nrows + RPB - 1) / RPB)), dim3(256), 0, L.stream, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? SIA_OK : fail(SIA_ERR_LAUNCH, "scored prefill launch: %s", hipGetErrorString(e));
}

template <int D, class T, int VAR>
static int launch_scored_var(PrefillLaunch& L) {
  switch (L.mod) {
    case kModMask: return launch_scored_mod<D, T, VAR, kModMask>(L);
    case kModCap: return launch_scored_mod<D, T, VAR, kModCap>(L);
    case kModBias: return launch_scored_mod<D, T, VAR, kModBias>(L);
    default: return launch_scored_mod<D, T, VAR, kModCapBias>(L);
  }
}

template <int D, class T>
static int launch_scored_typed(PrefillLaunch& L) {
  if (L.pack.nblocks > 0)
    hipLaunchKernelGGL((prefill_pack_v<D, T, true>), dim3((unsigned)L.pack.nblocks), dim3(256), 0, L.stream, L.pack);
  if constexpr ((D == 32 || D == 64 || D == 128) && std::is_same<T, BF16>::value)
    if (L.var == 2) return launch_scored_var<D, T, 2>(L);
  if constexpr (D == 128)
    if (L.var == 1) return launch_scored_var<D, T, 1>(L);
  if (L.var >= 3) return launch_prefill_scored_split(L);
  if (L.var != 0) return fail(SIA_ERR_LAUNCH, "prefill variant %d is not built for head_dim %d", L.var, D);
  return launch_scored_var<D, T, 0>(L);
}

template <int D>
static int launch_scored_d(PrefillLaunch& L) {
  return L.dtype == SIA_BF16 ? launch_scored_typed<D, BF16>(L) : launch_scored_typed<D, F16>(L);
}

}  // namespace sia
