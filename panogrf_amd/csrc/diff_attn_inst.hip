// The differential attention kernels of one direction, element type and head width (-DPGRF_DA_BWD, -DPGRF_DA_TYPE, -DPGRF_DA_D), and their launches.
#include "pgrf_experiments.h"
#include "diff_attn.h"

namespace pgrf {
namespace tok {

#if PGRF_DA_TYPE == 0
using DaT = float;
#elif PGRF_DA_TYPE == 1
using DaT = bf16;
#else
using DaT = f16;
#endif

#define PGRF_DA_NAME2(a, b, c) a##_##b##_##c
#define PGRF_DA_NAME1(a, b, c) PGRF_DA_NAME2(a, b, c)
#define PGRF_DA_NAME(f) PGRF_DA_NAME1(f, PGRF_DA_TYPE, PGRF_DA_D)

#if !PGRF_DA_BWD
template <int HOW>
static void launch_fwd(const DiffArgs& a, int waves, unsigned grid, hipStream_t s) {
  // (16 bits: up to 32 rows, one wave or a pair of them, are kTwo; kInF16 is for whole workgroups of rows)
  constexpr int D = PGRF_DA_D;
  constexpr bool few = (HOW == kTwo) == (PGRF_DA_TYPE != 0), whole = HOW == kInF16;
  if constexpr (D < 128 && few) {
    if (waves == 1) hipLaunchKernelGGL((diff_attn_fwd<DaT, D, 1, HOW>), dim3(grid), dim3(64), 0, s, a);
  }
  if constexpr ((D < 128 && !whole) || few) {
    if (waves == 2) hipLaunchKernelGGL((diff_attn_fwd<DaT, D, 2, HOW>), dim3(grid), dim3(128), 0, s, a);
  }
  if constexpr (D < 128 || !whole) {
    if (waves == 4) hipLaunchKernelGGL((diff_attn_fwd<DaT, D, 4, HOW>), dim3(grid), dim3(256), 0, s, a);
  }
  if constexpr (D == 128 && PGRF_DA_TYPE != 0) {
    if (waves == 8) hipLaunchKernelGGL((diff_attn_fwd<DaT, D, 8, HOW>), dim3(grid), dim3(512), 0, s, a);
  }
}

int PGRF_DA_NAME(launch_da_fwd)(const DiffArgs& a, int waves, unsigned grid, int how, hipStream_t s) {
  const char* who = "pgrf_diff_attention";
#if PGRF_DA_TYPE == 0
  launch_fwd<kOne>(a, waves, grid, s);
#else
  if (how == kOne) launch_fwd<kOne>(a, waves, grid, s);
#if PGRF_DA_TYPE == 1
  if (how == kInF16) {
    const dim3 parts((unsigned)(a.B * a.Hk * a.v_parts));
    hipLaunchKernelGGL((diff_attn_v_sizes<DaT, PGRF_DA_D>), parts, dim3(256), 0, s, a);
    PGRF_TOK_LAUNCHED(who);
    hipLaunchKernelGGL((diff_attn_v16<DaT, PGRF_DA_D>), parts, dim3(256), 0, s, a);
    PGRF_TOK_LAUNCHED(who);
    launch_fwd<kInF16>(a, waves, grid, s);
    PGRF_TOK_LAUNCHED(who);
  }
#endif
  if (how != kOne) launch_fwd<kTwo>(a, waves, grid, s);                        // (behind kInF16: the key heads that it left)
#endif
  PGRF_TOK_LAUNCHED(who);
  if (a.splits > 1) {
    const long long rows = (long long)a.B * a.Hk * a.N * a.G, per = 256 / (2 * PGRF_DA_D);
    constexpr int S = 1024 / (2 * PGRF_DA_D);
    if (a.splits > 8) hipLaunchKernelGGL((diff_attn_join<DaT, PGRF_DA_D, S>), dim3((unsigned)rows), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((diff_attn_join<DaT, PGRF_DA_D, 1>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a);
    PGRF_TOK_LAUNCHED(who);
  }
  return PGRF_OK;
}

#else
template <int NW>
static void launch_dkv(const DiffArgs& a, unsigned grid, hipStream_t s) {
  if constexpr (PGRF_DA_D == 128) {
    hipLaunchKernelGGL((diff_attn_dkv<DaT, PGRF_DA_D, NW, false, true>), dim3(grid), dim3(NW * 64), 0, s, a);
    hipLaunchKernelGGL((diff_attn_dkv<DaT, PGRF_DA_D, NW, true, false>), dim3(grid), dim3(NW * 64), 0, s, a);
  } else {
    hipLaunchKernelGGL((diff_attn_dkv<DaT, PGRF_DA_D, NW, true, true>), dim3(grid), dim3(NW * 64), 0, s, a);
  }
}

int PGRF_DA_NAME(launch_da_bwd)(const DiffArgs& a, int row_waves, unsigned row_grid, int units, int key_waves, unsigned key_grid, hipStream_t s) {
  const char* who = "pgrf_diff_attention_backward";
  auto lams = [&]() { hipLaunchKernelGGL((diff_attn_dlam<DaT>), dim3(a.H), dim3(1024), 0, s, a, units); };
#if PGRF_DA_D == 32 || (PGRF_DA_D == 64 && PGRF_DA_TYPE != 0)
  if (row_waves == 0) {
    if (key_waves == 1) hipLaunchKernelGGL((diff_attn_short<DaT, PGRF_DA_D, 1>), dim3(key_grid), dim3(64), 0, s, a);
    else hipLaunchKernelGGL((diff_attn_short<DaT, PGRF_DA_D, 2>), dim3(key_grid), dim3(128), 0, s, a);
    PGRF_TOK_LAUNCHED(who);
    if (a.dlam) {
      lams();
      PGRF_TOK_LAUNCHED(who);
    }
    return PGRF_OK;
  }
#endif
#if PGRF_DA_TYPE == 2
  const long long parts = (long long)a.B * a.Hk * a.size_parts;
  hipLaunchKernelGGL((diff_attn_sizes<DaT, PGRF_DA_D>), dim3((unsigned)(parts < (1 << 16) ? parts : 1 << 16)), dim3(256), 0, s, a);
  PGRF_TOK_LAUNCHED(who);
#endif
  if (row_waves == 1) hipLaunchKernelGGL((diff_attn_dq<DaT, PGRF_DA_D, 1>), dim3(row_grid), dim3(64), 0, s, a);
  else if (row_waves == 2) hipLaunchKernelGGL((diff_attn_dq<DaT, PGRF_DA_D, 2>), dim3(row_grid), dim3(128), 0, s, a);
  else hipLaunchKernelGGL((diff_attn_dq<DaT, PGRF_DA_D, 4>), dim3(row_grid), dim3(256), 0, s, a);
  PGRF_TOK_LAUNCHED(who);
  auto add = [&](const float* part, void* out, long long n, int shares) {
    hipLaunchKernelGGL((diff_attn_add<DaT>), dim3((unsigned)(n / 1024 < 2048 ? n / 1024 + 1 : 2048)), dim3(256), 0, s, part, (DaT*)out, n, shares);
  };
  if (a.dq && a.q_shares > 1) {
    add(a.dq_part, a.dq, (long long)a.B * a.N * a.H * 2 * PGRF_DA_D, a.q_shares);
    PGRF_TOK_LAUNCHED(who);
  }
  if (a.dlam) {
    lams();
    PGRF_TOK_LAUNCHED(who);
  }
  if (a.dk) {
    if (key_waves == 1) launch_dkv<1>(a, key_grid, s);
    else if (key_waves == 2) launch_dkv<2>(a, key_grid, s);
    else launch_dkv<4>(a, key_grid, s);
    PGRF_TOK_LAUNCHED(who);
    if (a.kv_shares > 1) {
      add(a.dk_part, a.dk, (long long)a.B * a.M * a.Hk * 2 * PGRF_DA_D, a.kv_shares);
      add(a.dv_part, a.dv, (long long)a.B * a.M * a.Hk * 2 * PGRF_DA_D, a.kv_shares);
      PGRF_TOK_LAUNCHED(who);
    }
  }
  return PGRF_OK;
}

#endif

}  // namespace tok
}  // namespace pgrf
