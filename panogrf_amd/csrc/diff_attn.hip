// C entries of the differential attention: checks, the cut of the work, and the choice of the kernels (diff_attn.h).
#include "pgrf_experiments.h"
#include "diff_attn.h"

namespace pgrf {
namespace tok {

#define PGRF_DA_DECL(T, D)                                                                       \
  int launch_da_fwd_##T##_##D(const DiffArgs& a, int waves, unsigned grid, int how, hipStream_t s); \
  int launch_da_bwd_##T##_##D(const DiffArgs& a, int row_waves, unsigned row_grid, int units, int key_waves, unsigned key_grid, hipStream_t s);
#define PGRF_DA_ALL(X) X(0, 32) X(0, 64) X(0, 128) X(1, 32) X(1, 64) X(1, 128) X(2, 32) X(2, 64) X(2, 128)
PGRF_DA_ALL(PGRF_DA_DECL)

static int waves_for(long long rows) { return rows > 64 ? 4 : rows > 32 ? 2 : 1; }

// The forward kernel's waves and their rows: at D = 128 two waves share 32 rows (and float's values leave no room for eight)
struct FwdCut { int waves, rows, splits, how, v_parts; };
static FwdCut cut_fwd(int dtype, int B, int Hk, long long rows, int M, int D) {
  FwdCut f;
  // (kTwo, kInF16 and what they cost stand at their names.  v in f16 from 2^33 products of a score and 1024 rows on: a forward pass there takes 100-180 us and 12-20 more with the
  // launches over v, at 2^34 11 or 23 more on 220, at 2^32 17 on 67 and 12 on 101; 64 x 512 rows and keys, 2^33: 45 more on 176.)
  f.how = dtype == PGRF_DTYPE_F32 ? kOne : rows <= 32 || M <= 64 ? kTwo : dtype == PGRF_DTYPE_BF16 && rows >= 1024 && (double)B * Hk * rows * M * D >= 8589934592.0 ? kInF16 : kOne;
  f.v_parts = f.how != kInF16 ? 0 : M > 256 * 64 ? 256 : (M + 63) / 64;
  f.waves = waves_for(rows);
  if (D == 128) f.waves = f.waves == 4 && dtype == PGRF_DTYPE_F32 ? 4 : 2 * f.waves;
  f.rows = D == 128 ? f.waves * 16 : f.waves * 32;
  const long long groups = (long long)B * Hk * ((rows + f.rows - 1) / f.rows);
  // The key axis is cut where the rows alone leave the chip idle.  Up to 32 rows (single tokens) it is dealt out to five workgroups of one wave for every CU; more of them
  // cost more in partial sums than they even out (32 caches of 4096 to 16384 keys, 8 key heads, bf16, D = 64: 245 us; with 1024 263, with 2560 257, with 5120 285).  There a
  // share may be a single block of 32 keys, as a wave's blocks come one after the other (one cache of 500 keys, 2 key heads: 10.5 us; with 64 keys at least 11.0, with
  // 128 15.7).  More rows: 512 workgroups fit, and from half of that on the join costs more than the idle half (2048 x 8192, 16 heads: 245 us whole, 271 cut).
  const bool few = rows <= 32;
  const long long want = few ? 1280 : 512, most = few ? (M + 31) / 32 : M / 128;
  long long s = !few && groups > want / 2 ? 1 : (want + groups - 1) / groups;
  if (s > most) s = most;
  if (s > 128) s = 128;
  f.splits = s < 1 ? 1 : (int)s;
  return f;
}

// The backward kernels' waves, workgroups and shares.  The chip holds 512 workgroups of four waves at a time (256 where their registers or tiles leave room for one per
// CU).  Where there are fewer, or where the causal mask makes some twice as long as the mean and they cannot be dealt out, a workgroup's blocks are cut into shares of at
// least 8 whose gradients are added in float behind.
struct BwdCut { int row_waves, key_waves, q_shares, kv_shares, units; long long row_groups, key_groups; };
static int shares_for(long long groups, long long blocks, bool causal, int places) {
  const long long want = causal ? 2 * places : places;
  if (groups * 4 > want * 3) return 1;
  long long s = (want + groups - 1) / groups;
  if (s > blocks / 8) s = blocks / 8;
  return (int)(s > 16 ? 16 : s < 1 ? 1 : s);
}
static BwdCut cut_bwd(int dtype, int B, int N, int M, int H, int Hk, int D, bool causal) {
  BwdCut c;
  const int G = H / Hk, places = dtype == PGRF_DTYPE_F32 || D == 128 ? 256 : 512;
  const long long rows = (long long)N * G;
  // Key heads with up to 64 keys, as long as there is one for every CU: a workgroup each forms all gradients (row_waves 0).  (float, D = 32, 64 keys: 2048 rays of 4 heads x
  // 64 samples 351 us, with the two kernels 523; 256 key heads x 2048 queries 400, 512; 128 of them 404, 270.  At D = 64 float's values fill the registers: 535 both ways.)
  if (M <= 64 && D * (int)dtype_bytes(dtype) <= 128 && (long long)B * Hk >= 256) return {0, M > 32 ? 2 : 1, 1, 1, 1, 0, (long long)B * Hk};
  c.row_waves = waves_for(rows);
  c.key_waves = waves_for(M);
  c.row_groups = (long long)B * Hk * ((rows + c.row_waves * 32 - 1) / (c.row_waves * 32));
  c.key_groups = (long long)B * Hk * (((long long)M + c.key_waves * 32 - 1) / (c.key_waves * 32));
  // (short key axes form delta in a sweep of their own, which every share would repeat)
  c.q_shares = M < 1024 ? 1 : shares_for(c.row_groups, (M + 31) / 32, causal, places);
  c.kv_shares = shares_for(c.key_groups, (long long)G * ((N + 31) / 32), causal, places);
  // (a wave's parts of dlam: G for 32 rows, rounded up to whole workgroups of at most four waves; fewer than N + 4 of each head)
  c.units = ((G & (G - 1)) == 0 && G <= 32 ? (int)((rows + c.row_waves * 32 - 1) / (c.row_waves * 32) * c.row_waves) : N) * c.q_shares;
  return c;
}

// Workgroups that look for a key head's largest values (f16)
static int size_parts(int dtype, int N, int M, int G) {
  if (dtype != PGRF_DTYPE_F16) return 0;
  const long long most = (long long)N * G > M ? (long long)N * G : M;
  return most > 256 * 64 ? 256 : (int)((most + 63) / 64);
}

// Whether a launch has room for so many workgroups: 2^32 - 1 threads.  With B Hk below 2^25, and B H N and (for gradients) B Hk M below 2^29, all launches do: up to 64 rows or
// keys a key head takes 128 threads, beyond that a row or key less than eight.
static bool fits(long long workgroups, int threads) { return workgroups <= 0x7fffffffll && workgroups * threads <= 0xffffffffll; }

static int check(const PgrfDiffAttn* p, const char* who, bool backward) {
  if (!p) return set_error(PGRF_ERR_ARG, "%s: null arguments", who);
  if (!dtype_ok(p->dtype)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: dtype %d (PGRF_DTYPE_F32 | BF16 | F16)", who, p->dtype);
  if (p->D != 32 && p->D != 64 && p->D != 128) return set_error(PGRF_ERR_UNSUPPORTED, "%s: D=%d (32, 64 or 128)", who, p->D);
  if (p->B < 0 || p->N < 0 || p->M < 1 || p->H < 1 || p->Hk < 1 || p->H % p->Hk)
    return set_error(PGRF_ERR_ARG, "%s: bad sizes B=%d N=%d M=%d H=%d Hk=%d (H a multiple of Hk, M at least 1)", who, p->B, p->N, p->M, p->H, p->Hk);
  if (!(p->scale > 0.f) || p->scale > 1e30f) return set_error(PGRF_ERR_ARG, "%s: scale must be positive", who);
  if ((long long)p->N * (p->H / p->Hk) > 0x3fffffff || (long long)p->B * p->N > 0x3fffffff || p->M > 0x3fffffff)
    return set_error(PGRF_ERR_UNSUPPORTED, "%s: over 2^30 rows", who);
  if ((long long)p->B * p->Hk > (1 << 26)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: too many tiles", who);   // (what is counted from here on fits 64 bits)
  if ((long long)p->B * p->N == 0) return PGRF_OK;
  if (!p->q || !p->k || !p->v || !p->lam) return set_error(PGRF_ERR_ARG, "%s: null q / k / v / lam", who);
  const long long per = 16 / (long long)dtype_bytes(p->dtype);
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) ||
      (p->q_sb | p->q_sn | p->q_sh | p->q_sm | p->k_sb | p->k_sn | p->k_sh | p->k_sm | p->v_sb | p->v_sn | p->v_sh) % per)
    return set_error(PGRF_ERR_ARG, "%s: q, k, v: addresses and strides must be multiples of 16 bytes", who);
  // (what a tile's lanes add to its base has to fit 32 bits; nothing is added for an axis of one token)
  auto far = [](long long stride) { return stride < 0 || stride > (1 << 22); };
  if ((p->N > 1 && far(p->q_sn)) || far(p->q_sm) || (p->M > 1 && (far(p->k_sn) || far(p->v_sn))) || far(p->k_sm) || (long long)p->H * 2 * p->D > (1 << 22))
    return set_error(PGRF_ERR_UNSUPPORTED, "%s: a stride between tokens or maps is negative or over 2^22 values", who);
  if (backward && !p->lse) return set_error(PGRF_ERR_ARG, "%s: null lse", who);
  if (backward && p->lengths) return set_error(PGRF_ERR_UNSUPPORTED, "%s: lengths have no backward pass (use key_mask)", who);
  if (!backward && !p->out) return set_error(PGRF_ERR_ARG, "%s: null out", who);
  if (!p->lse && p->maps_out) return set_error(PGRF_ERR_ARG, "%s: maps_out without lse", who);
  if ((p->maps_out && !aligned16(p->maps_out)) || (p->out && !aligned16(p->out))) return set_error(PGRF_ERR_ARG, "%s: out / maps_out must be 16-byte aligned", who);
  return PGRF_OK;
}

static DiffArgs args_of(const PgrfDiffAttn* p) {
  DiffArgs a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.lam = p->lam;
  a.q_sb = p->q_sb; a.q_sn = p->q_sn; a.q_sh = p->q_sh; a.q_sm = p->q_sm;
  a.k_sb = p->k_sb; a.k_sn = p->k_sn; a.k_sh = p->k_sh; a.k_sm = p->k_sm;
  a.v_sb = p->v_sb; a.v_sn = p->v_sn; a.v_sh = p->v_sh;
  a.mask = p->key_mask; a.mask_sb = p->mask_sb; a.lengths = p->lengths;
  a.B = p->B; a.N = p->N; a.M = p->M; a.H = p->H; a.Hk = p->Hk; a.G = p->H / p->Hk; a.causal = p->causal ? 1 : 0; a.lam_f32 = p->lam_f32 ? 1 : 0;
  a.scale = p->scale; a.c = p->scale * kLog2e;
  a.out = p->out; a.lse = p->lse; a.o12 = p->maps_out; a.splits = 1;
  return a;
}

}  // namespace tok
}  // namespace pgrf

using namespace pgrf;
using namespace pgrf::tok;

extern "C" {

size_t pgrf_diff_attention_workspace_bytes(int dtype, int B, int N, int M, int H, int Hk, int D) {
  if (B < 1 || N < 1 || M < 1 || H < 1 || Hk < 1 || H % Hk || D < 1) return 0;
  const long long rows = (long long)N * (H / Hk);
  const FwdCut c = cut_fwd(dtype, B, Hk, rows, M, D);
  size_t n = c.splits > 1 ? (size_t)c.splits * B * Hk * rows * (4 * D + 4) * sizeof(float) : 0;
  if (c.how == kInF16) n += (size_t)B * Hk * M * 2 * D * 2 + ((size_t)B * Hk * c.v_parts * 8 + 15) / 16 * 16 + ((size_t)B * Hk * 4 + 15) / 16 * 16;
  return n;
}

int pgrf_diff_attention(const PgrfDiffAttn* p, void* stream) {
  const char* who = "pgrf_diff_attention";
  int rc = check(p, who, false);
  if (rc) return rc;
  if ((long long)p->B * p->N == 0) return PGRF_OK;
  DiffArgs a = args_of(p);
  const long long rows = (long long)a.N * a.G;
  const FwdCut cut = cut_fwd(p->dtype, a.B, a.Hk, rows, a.M, p->D);
  a.splits = cut.splits;
  const size_t need = pgrf_diff_attention_workspace_bytes(p->dtype, p->B, p->N, p->M, p->H, p->Hk, p->D);
  if (need && (!p->workspace || !aligned16(p->workspace) || p->workspace_bytes < need))
    return set_error(PGRF_ERR_ARG, "%s: workspace too small or not 16-byte aligned (%zu < %zu bytes)", who, p->workspace_bytes, need);
  char* room = (char*)p->workspace;
  if (a.splits > 1) {
    const size_t n = (size_t)a.splits * a.B * a.Hk * rows;
    a.part_o = (float*)room;
    a.part_ml = a.part_o + n * 4 * p->D;
    room += n * (4 * p->D + 4) * sizeof(float);
  }
  if (cut.how == kInF16) {
    a.v_parts = cut.v_parts;
    a.v16 = room;
    room += (size_t)a.B * a.Hk * a.M * 2 * p->D * 2;
    a.v_sizes = (float*)room;
    a.v_exp = (int*)(room + ((size_t)a.B * a.Hk * a.v_parts * 8 + 15) / 16 * 16);
  }
  const long long grid = (long long)a.B * a.Hk * ((rows + cut.rows - 1) / cut.rows) * a.splits;
  if (!fits(grid, cut.waves * 64) || !fits((long long)a.B * a.Hk * cut.v_parts, 256)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: too many tiles", who);
#define PGRF_DA_FWD(T, D_) \
  if (p->dtype == T && p->D == D_) return launch_da_fwd_##T##_##D_(a, cut.waves, (unsigned)grid, cut.how, (hipStream_t)stream);
  PGRF_DA_ALL(PGRF_DA_FWD)
  return set_error(PGRF_ERR_UNSUPPORTED, "%s: no kernel", who);
}

int pgrf_diff_attention_keeps_maps(int dtype, int M) { return M > (dtype == PGRF_DTYPE_F32 ? 64 : 512); }

size_t pgrf_diff_attention_backward_workspace_bytes(int dtype, int B, int N, int M, int H, int Hk, int D, int causal) {
  if (B < 1 || N < 1 || M < 1 || H < 1 || Hk < 1 || H % Hk || D < 1) return 0;
  const BwdCut c = cut_bwd(dtype, B, N, M, H, Hk, D, causal != 0);
  size_t n = (size_t)B * H * 2 * N + ((size_t)B * Hk * c.units * (H / Hk) + 3) / 4 * 4;
  n = (n + 3) / 4 * 4;
  if (c.row_waves) n += ((size_t)B * Hk * size_parts(dtype, N, M, H / Hk) * 2 + 3) / 4 * 4;
  if (c.q_shares > 1) n += (size_t)c.q_shares * B * N * H * 2 * D;
  if (c.kv_shares > 1) n += (size_t)c.kv_shares * B * M * Hk * 4 * D;
  return n * sizeof(float);
}

int pgrf_diff_attention_backward(const PgrfDiffAttn* p, const void* dout, void* dq, void* dk, void* dv, void* dlam, void* stream) {
  const char* who = "pgrf_diff_attention_backward";
  int rc = check(p, who, true);
  if (rc) return rc;
  if (!dk != !dv) return set_error(PGRF_ERR_ARG, "%s: dk and dv go together", who);
  if ((long long)p->B * p->N == 0) return set_error(PGRF_ERR_ARG, "%s: no rows: the gradients are 0", who);
  if (!dout || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return set_error(PGRF_ERR_ARG, "%s: dout null, or a tensor not 16-byte aligned", who);
  const BwdCut c = cut_bwd(p->dtype, p->B, p->N, p->M, p->H, p->Hk, p->D, p->causal != 0);
  const long long rg = c.row_groups * c.q_shares, kg = c.key_groups * c.kv_shares;
  if (!fits(rg, c.row_waves * 64) || !fits(kg, c.key_waves * 64)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: too many tiles", who);
  const size_t need = pgrf_diff_attention_backward_workspace_bytes(p->dtype, p->B, p->N, p->M, p->H, p->Hk, p->D, p->causal);
  if (!p->workspace || !aligned16(p->workspace) || p->workspace_bytes < need)
    return set_error(PGRF_ERR_ARG, "%s: workspace too small or not 16-byte aligned (%zu < %zu bytes)", who, p->workspace_bytes, need);
  DiffArgs a = args_of(p);
  a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv; a.dlam = dlam;
  a.delta = (float*)p->workspace;
  a.q_shares = c.q_shares; a.kv_shares = c.kv_shares;
  const size_t sums = (size_t)a.B * a.H * 2 * a.N;
  a.dlam_part = a.delta + sums;
  float* behind = a.delta + (sums + ((size_t)a.B * a.Hk * c.units * a.G + 3) / 4 * 4 + 3) / 4 * 4;
  if (c.row_waves) {
    a.size_parts = size_parts(p->dtype, a.N, a.M, a.G);
    a.sizes = behind;
    behind += ((size_t)a.B * a.Hk * a.size_parts * 2 + 3) / 4 * 4;
  }
  if (c.q_shares > 1) { a.dq_part = behind; behind += (size_t)c.q_shares * a.B * a.N * a.H * 2 * p->D; }
  if (c.kv_shares > 1) { a.dk_part = behind; a.dv_part = behind + (size_t)c.kv_shares * a.B * a.M * a.Hk * 2 * p->D; }
#define PGRF_DA_BWD(T, D_) \
  if (p->dtype == T && p->D == D_) return launch_da_bwd_##T##_##D_(a, c.row_waves, (unsigned)rg, c.units, c.key_waves, (unsigned)kg, (hipStream_t)stream);
  PGRF_DA_ALL(PGRF_DA_BWD)
  return set_error(PGRF_ERR_UNSUPPORTED, "%s: no kernel", who);
}

}  // extern "C"
