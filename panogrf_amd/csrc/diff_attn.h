// Differential attention: out = (A1 - lam A2) v with two softmax maps A_i = softmax(scale q_i k_i^T + mask), forward and backward.
//
// Shapes.  q [B,N,H,2,D], k [B,M,Hk,2,D], v [B,M,Hk,2D], lam [H]; G = H / Hk query heads share a key head.  The rows of a key head are its
// N G (token, head) pairs, token first, so that query heads that share keys also share the tiles that hold them, and a single token of G heads fills
// one tile of rows.
//
// Tiles.  Products run on 32x32 matrix instructions with float accumulators.  One wave owns 32 rows (forward, dq) or 32 keys (dk, dv); the other side passes
// through LDS in tiles that all waves of a workgroup read.  Every score block is formed transposed to how it is used next: S^T = K Q^T leaves a lane with 16 keys of
// ONE row (the other 16 in lane ^ 32), so softmax sums need one exchange, the rescaling of a row is a scalar of its lane, and the 8 values that a
// lane holds for 16 consecutive keys are already an operand of the next product, if that product counts its keys in the order 0-3, 8-11 | 4-7, 12-15.
// The other operand follows that order by which rows it reads (mm.tr below).
#pragma once
#include "token_common.h"

namespace pgrf {
namespace tok {

using f32x16 = __attribute__((ext_vector_type(16))) float;

// 32x32 products.  A fragment is 8 values of one row of A (or column of B): lane l holds row l & 31, places 8 (l >> 5) .. + 7 of a step of 16.
template <typename T> struct Frag8 { typedef T type __attribute__((ext_vector_type(8))); };

__device__ __forceinline__ f32x16 mma(Frag8<bf16>::type a, Frag8<bf16>::type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(Frag8<f16>::type a, Frag8<f16>::type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// float: eight products of two places each; which place of the step they take is the same for both operands, so its order does not matter
__device__ __forceinline__ f32x16 mma(Frag8<float>::type a, Frag8<float>::type b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// A tile of rows of 2 D values in LDS, in chunks of 16 bytes; chunk c of row r lies at place c ^ turn(r).  Reading the same chunk of 8 consecutive rows, or two
// neighbouring chunks of 4, meets every bank once.
template <typename T, int D>
struct Tile {
  static constexpr int kRow = 2 * D * (int)sizeof(T), kChunks = kRow / 16, kPer = 16 / (int)sizeof(T);
  using F = typename Frag8<T>::type;
  static __device__ __forceinline__ int turn(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }
  static __device__ __forceinline__ const char* at(const char* t, int r, int c) { return t + r * kRow + ((c ^ turn(r)) << 4); }

  // 8 values from value e (a multiple of 8) of row r
  static __device__ __forceinline__ F row(const char* t, int r, int e) {
    if constexpr (sizeof(T) == 2) {
      return *(const F*)at(t, r, e / 8);
    } else {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const f4 lo = *(const f4*)at(t, r, e / 4), hi = *(const f4*)at(t, r, e / 4 + 1);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // the transposed fragment: value e0 + (lane & 31) of rows r0 + 4 h + {0..3, 8..11}, h = lane >> 5
  static __device__ __forceinline__ F col(const char* t, int r0, int e0, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr: the 16 lanes of a group hand in 4 rows x 16 values (4 values each) and each gets a column of 4
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const int i = lane & 15, e = e0 + (lane & 16) + (i & 3) * 4, r = r0 + 4 * h + (i >> 2);
      const char* p = at(t, r, e / 8) + (i & 1) * 8;
      const char* q = at(t, r + 8, e / 8) + (i & 1) * 8;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(__attribute__((address_space(3))) char*)p);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(__attribute__((address_space(3))) char*)q);
      const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(F, v);
    } else {
      const int e = e0 + (lane & 31);
      F v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = r0 + 4 * h + (j & 3) + (j >> 2) * 8;
        v[j] = *(const float*)(at(t, r, e / 4) + (e & 3) * 4);
      }
      return v;
    }
  }
  // Brings R rows of a strided matrix (two halves of D values, `sm` apart) into a tile, without registers.  What a lane fetches in a tile is fixed: step i of its wave
  // is row `row(i)`, value `val(i)`; only the uniform base moves from tile to tile.
  template <int R, int NW>
  struct Loader {
    static constexpr int kSteps = R * kChunks / 64 / NW, kRowsPer = 64 * NW / kChunks;   // rows between a lane's steps
    static_assert(R * kChunks % (64 * NW) == 0 && kRowsPer * kChunks == 64 * NW, "whole waves, whole rows");
    int row0, sn, sm;
    __device__ Loader(long long sn_, long long sm_, int tid) : row0(tid / kChunks), sn((int)sn_), sm((int)sm_) {}
    __device__ __forceinline__ int val(int i, int tid) const {
      const int e = ((tid % kChunks) ^ turn(row0 + i * kRowsPer)) * kPer;
      return e >= D ? e - D + sm : e;
    }
    // base: the tile's first row; rows from `rows` on repeat the last one (they are masked)
    __device__ __forceinline__ void operator()(char* t, const T* base, int rows, int tid, int wave) const {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int r = row0 + i * kRowsPer, g = min(r, rows - 1);
        const char* p = (const char*)base + (unsigned)((g * sn + val(i, tid)) * (int)sizeof(T));
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)(t + (i * NW + wave) * 1024), 16, 0, 0);
      }
    }
  };
  // rows whose bit is not set in `keep` are set to zero
  template <int R, int THREADS>
  static __device__ __forceinline__ void clear(char* t, unsigned long long keep, int tid) {
    for (int i = tid; i < R * kChunks; i += THREADS)
      if (!((keep >> (i / kChunks)) & 1)) *(float4*)(t + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
};

struct DiffArgs {
  const void *q, *k, *v, *lam;
  long long q_sb, q_sn, q_sh, q_sm, k_sb, k_sn, k_sh, k_sm, v_sb, v_sn, v_sh;
  const unsigned char* mask;      // [B,M] by mask_sb: 0 = no query sees the key
  long long mask_sb;
  const int* lengths;             // [B]: keys of each batch entry that count (NULL: M)
  int B, N, M, H, Hk, G, causal, lam_f32;
  float c, scale;                 // c = scale * log2(e): probabilities are powers of two
  void* out;                      // [B,N,H,2D]
  float* lse;                     // [B,H,2,N]: log2 of the sum behind each map, +inf where a row sees nothing
  float* o12;                     // [B,N,H,2,2D]: the two maps' outputs
  // a key axis cut into `splits`: partial [splits][B*Hk][N*G] rows of 2 x 2D values and (m1, l1, m2, l2)
  int splits;
  float *part_o, *part_ml;
  // backward
  const void* dout;               // [B,N,H,2D] contiguous
  float* delta;                   // [B,H,2,N]: dout . o_i
  float* dlam_rows;               // [B,H,N]
  void *dq, *dk, *dv, *dlam;
};

constexpr float kLog2e = 1.44269504088896340736f;

// Workgroups go round the 8 XCDs one by one; this gives each XCD a contiguous share, so that workgroups of one key head read it through one L2.
__device__ __forceinline__ unsigned by_xcd(unsigned id, unsigned n) {
  const unsigned per = n / 8, rest = n % 8, x = id % 8, i = id / 8;
  return x < rest ? x * (per + 1) + i : rest * (per + 1) + (x - rest) * per + i;
}

template <typename T>
__device__ __forceinline__ float lam_of(const DiffArgs& a, int h) {
  return a.lam_f32 ? ((const float*)a.lam)[h] : (float)((const T*)a.lam)[h];
}

template <typename T>
__device__ __forceinline__ typename Frag8<T>::type pack(const f32x16& p, int s) {   // values 8 s .. 8 s + 7
  typename Frag8<T>::type v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)p[8 * s + j];
  return v;
}

template <typename T>
__device__ __forceinline__ typename Frag8<T>::type load8(const T* p) {
  if constexpr (sizeof(T) == 2) {
    return *(const typename Frag8<T>::type*)p;
  } else {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 lo = *(const f4*)p, hi = *(const f4*)(p + 4);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// row of a 32x32 accumulator: value r of lane l is (row_of(r, l >> 5), column l & 31)
__device__ __forceinline__ constexpr int row_of(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  Vec<T, 4> v;
  v.e[0] = (T)a; v.e[1] = (T)b; v.e[2] = (T)c; v.e[3] = (T)d;
  store_vec<T, 4>(p, v);
}

// Which keys of the R keys from k0 any query may see: bit r = key k0 + r (uniform over the workgroup)
template <int R>
__device__ __forceinline__ unsigned long long keys_seen(const unsigned char* mask, int k0, int len, int lane) {
  const int k = k0 + lane;
  const bool in = lane < R && k < len && (!mask || mask[k]);
  return __ballot(in);
}

// Bit row_of(i, 0): whether value i of a lane, key row_of(i, h) of its block, counts for a row whose last key is `last` keys behind the block's first
__device__ __forceinline__ unsigned keys_of_lane(unsigned seen32, int last, int h) {
  const unsigned upto = last >= 31 ? ~0u : last < 0 ? 0u : (2u << last) - 1;
  return (seen32 & upto) >> (4 * h);
}

// ---------------------------------------------------------------------------------------------------------------- forward
// MPW: maps of a wave.  Up to D = 64 a wave keeps the sums of both maps of its 32 rows (128 registers), and every fragment of v serves two products.  At
// D = 128 two waves share 32 rows, one map each, and meet at the end.
template <typename T, int D, int NW> struct FwdShape {
  static constexpr int MPW = D == 128 && NW > 1 ? 1 : 2;
  static constexpr int KT = 32;                                                // keys of a block
};

// Scores of a block: S^T of MPW maps
template <typename T, int D, int MPW>
__device__ __forceinline__ void scores(f32x16 (&s)[MPW], const char* kt, const typename Frag8<T>::type (&qf)[MPW][D / 16], int map0, int lane) {
#pragma unroll
  for (int m = 0; m < MPW; ++m) s[m] = zero16();
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int m = 0; m < MPW; ++m) s[m] = mma(Tile<T, D>::row(kt, lane & 31, (map0 + m) * D + 16 * i + 8 * (lane >> 5)), qf[m][i], s[m]);
}

__device__ __forceinline__ float top_of(const f32x16& s) {
  float t = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) t = fmaxf(t, s[i]);
  return t;
}
__device__ __forceinline__ float with_other_half(float t) {                    // the larger of lane and lane ^ 32
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// One pass over the keys in blocks of 32, three blocks in work at a time: while block j goes through its exponentials, the matrix pipe forms the scores of
// block j + 1 and adds block j - 1 times its values.  None of the three waits for another, and they stand in one stretch of code without a branch, so that a
// wave by itself keeps both pipes busy (measured on this card: 24 products of 32x32x16, 96 FMAs and 32 exponentials take 471 ns side by side, 386 + 312 one
// after the other); masks and a new maximum are dealt with in front of it.
#define PGRF_DA_WEAVE_FWD
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, (NW + 3) / 4) void diff_attn_fwd(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  using Sh = FwdShape<T, D, NW>;
  constexpr int KT = Sh::KT, MPW = Sh::MPW, NK = D / 16, NC = 2 * D / 32, RW = NW * MPW / 2;   // RW: groups of 32 rows in the workgroup
  constexpr int kTile = KT * TL::kRow;
  __shared__ __attribute__((aligned(16))) char tiles_lds[4 * kTile];             // two blocks of k, two of v
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int group = MPW == 2 ? wave : wave >> 1, map0 = MPW == 2 ? 0 : wave & 1;
  const int rows = a.N * a.G, tiles = (rows + RW * 32 - 1) / (RW * 32);
  unsigned id = by_xcd(blockIdx.x, gridDim.x);
  const int split = id % a.splits;
  id /= a.splits;
  const int tile = tiles - 1 - (int)(id % tiles);                              // (causal: the longest rows first)
  const int bh = id / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.M) : a.M;
  const int r0 = (tile * RW + group) * 32, r = r0 + (lane & 31), rc = min(r, rows - 1);
  const int n = rc / a.G, head = hk * a.G + rc % a.G;
  // the last key a row sees, of the wave's first row, and of the workgroup's last row
  const int off = len - a.N;
  const int lim = r >= rows ? -1 : a.causal ? min(n + off, len - 1) : len - 1;
  const int lim_lo = r0 + 31 >= rows ? -1 : a.causal ? min(r0 / a.G + off, len - 1) : len - 1;
  const int wg_hi = a.causal ? min(min((tile + 1) * RW * 32 - 1, rows - 1) / a.G + off, len - 1) : len - 1;
  const int all = (wg_hi + KT) / KT, per = (max(all, 0) + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(all, t0 + per);

  const T* q = (const T*)a.q + b * a.q_sb + n * a.q_sn + head * a.q_sh + map0 * a.q_sm + 8 * h;
  F qf[MPW][NK];
#pragma unroll
  for (int m = 0; m < MPW; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[m][s] = load8<T>(q + m * a.q_sm + 16 * s);

  const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
  const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const typename TL::template Loader<KT, NW> lk(a.k_sn, a.k_sm, tid), lv(a.v_sn, D, tid);
  auto ktile = [&](int t) { return tiles_lds + (t & 1) * kTile; };
  auto vtile = [&](int t) { return tiles_lds + 2 * kTile + (t & 1) * kTile; };
  auto fetch_k = [&](int t) { lk(ktile(t), k + (long long)t * KT * a.k_sn, len - t * KT, tid, wave); };
  auto fetch_v = [&](int t) { lv(vtile(t), v + (long long)t * KT * a.v_sn, len - t * KT, tid, wave); };

  f32x16 o[MPW][NC], s[MPW];
  F p[MPW][2];
  float mx[MPW], l[MPW], top[MPW];
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    mx[m] = -INFINITY;
    l[m] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[m][c] = zero16();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) p[m][i][j] = (T)0.f;
  }
  auto add_block = [&](const char* vt) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const F vf = TL::col(vt, 16 * i, 32 * c, lane);
#pragma unroll
        for (int m = 0; m < MPW; ++m) o[m][c] = mma(vf, p[m][i], o[m][c]);
      }
  };

  if (t0 < t1) {
    fetch_k(t0);
    for (int i = tid; i < kTile / 16; i += NW * 64) *(float4*)(vtile(t0 - 1) + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);   // (its probabilities are 0)
    unsigned seen = ~0u;
    __syncthreads();
    if (t0 + 1 < t1) fetch_k(t0 + 1);
    scores<T, D, MPW>(s, ktile(t0), qf, map0, lane);
#pragma unroll
    for (int m = 0; m < MPW; ++m) top[m] = top_of(s[m]);
    for (int t = t0; t < t1; ++t) {
      const int k0 = t * KT;
      const unsigned before = seen;
      seen = ~0u;
      if (mask || k0 + KT > len) seen = (unsigned)keys_seen<KT>(mask, k0, len, lane);
      __syncthreads();                                                         // k of t + 1 and v of t - 1 have come; nobody reads k of t or v of t - 2 any more
      if (t + 2 < t1) fetch_k(t + 2);
      if (before != ~0u) {                                                     // what stands in masked values may be anything, and 0 * NaN is NaN
        TL::template clear<KT, NW * 64>(vtile(t - 1), before, tid);
        __syncthreads();
      }
      fetch_v(t);
      if (seen != ~0u || k0 + 31 > lim_lo) {
        const unsigned ok = keys_of_lane(seen, lim - k0, h);
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[m][i] = (ok >> row_of(i, 0)) & 1 ? s[m][i] : -INFINITY;
          top[m] = top_of(s[m]);
        }
      }
      // The running maximum follows only where a row outgrew it by 2^8, and by a whole power of two: sums and values stay in range, and what was rounded before
      // scales without another rounding
#pragma unroll
      for (int m = 0; m < MPW; ++m) {
        const float up = with_other_half(top[m]) * a.c;
        if (__any(up > mx[m] + 8.f)) {
          const float grow = fmaxf(ceilf(up - mx[m]), 0.f), f = mx[m] == -INFINITY ? 1.f : ldexpf(1.f, -(int)fminf(grow, 1000.f));
          mx[m] = mx[m] == -INFINITY ? up : mx[m] + grow;
          l[m] *= f;
#pragma unroll
          for (int c = 0; c < NC; ++c) o[m][c] *= f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[m][i][j] = (T)((float)p[m][i][j] * f);
        }
      }
      f32x16 next[MPW];
      scores<T, D, MPW>(next, ktile(t + 1), qf, map0, lane);                   // (behind the last block: of whatever stands there, and unused)
      add_block(vtile(t - 1));
#pragma unroll
      for (int m = 0; m < MPW; ++m) {
        const float base = mx[m] == -INFINITY ? 0.f : mx[m];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[m][i] = __builtin_amdgcn_exp2f(fmaf(s[m][i], a.c, -base));
          sum += s[m][i];
        }
        l[m] += sum;
#pragma unroll
        for (int i = 0; i < 2; ++i) p[m][i] = pack<T>(s[m], i);
        s[m] = next[m];
        top[m] = top_of(s[m]);
      }
      PGRF_DA_WEAVE_FWD
    }
    __syncthreads();
    if (seen != ~0u) {
      TL::template clear<KT, NW * 64>(vtile(t1 - 1), seen, tid);
      __syncthreads();
    }
    add_block(vtile(t1 - 1));
  }
#pragma unroll
  for (int m = 0; m < MPW; ++m) l[m] += __shfl_xor(l[m], 32, 64);
  const bool live = r < rows;
  if (a.splits > 1) {
    if (!live) return;
    const long long at = ((long long)split * a.B * a.Hk + bh) * rows + r;
    float* po = a.part_o + at * 4 * D + map0 * 2 * D + 4 * h;
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<float>(po + m * 2 * D + 32 * c + 8 * g, o[m][c][4 * g], o[m][c][4 * g + 1], o[m][c][4 * g + 2], o[m][c][4 * g + 3]);
      if (h == 0) *(float2*)(a.part_ml + at * 4 + 2 * (map0 + m)) = make_float2(mx[m], l[m]);
    }
    return;
  }
  const float lam = lam_of<T>(a, head);
  const long long at = ((long long)b * a.N + n) * a.H + head;
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    const float inv = l[m] > 0.f ? 1.f / l[m] : l[m];                          // (a NaN stays one)
#pragma unroll
    for (int c = 0; c < NC; ++c) o[m][c] *= inv;
    if (a.o12 && live) {
      float* oo = a.o12 + at * 4 * D + (map0 + m) * 2 * D + 4 * h;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) store4<float>(oo + 32 * c + 8 * g, o[m][c][4 * g], o[m][c][4 * g + 1], o[m][c][4 * g + 2], o[m][c][4 * g + 3]);
      if (h == 0) a.lse[(((long long)b * a.H + head) * 2 + map0 + m) * a.N + n] = l[m] == 0.f ? INFINITY : mx[m] + log2f(l[m]);
    }
  }
  T* out = (T*)a.out + at * 2 * D + 4 * h;
  if constexpr (MPW == 1) {
    // the second map's waves hand their values over through LDS, as many column blocks at a time as the tiles' room holds
    constexpr int kFit = 4 * kTile / (RW * 64 * 64), kAt = kFit < NC ? kFit : NC;
    static_assert(kAt >= 1 && NC % kAt == 0, "");
    float* room = (float*)tiles_lds + group * kAt * 16 * 64 + lane;
    for (int c0 = 0; c0 < NC; c0 += kAt) {
      __syncthreads();                                                         // (also: the tiles are read)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (map0 == 1 && c >= c0 && c < c0 + kAt)
#pragma unroll
          for (int i = 0; i < 16; ++i) room[((c - c0) * 16 + i) * 64] = o[0][c][i];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (map0 == 0 && live && c >= c0 && c < c0 + kAt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = o[0][c][4 * g + j] - lam * room[((c - c0) * 16 + 4 * g + j) * 64];
            store4<T>(out + 32 * c + 8 * g, u[0], u[1], u[2], u[3]);
          }
    }
  } else {
    if (!live) return;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = o[0][c][4 * g + j] - lam * o[MPW - 1][c][4 * g + j];
        store4<T>(out + 32 * c + 8 * g, u[0], u[1], u[2], u[3]);
      }
  }
}

// Joins the shares of a cut key axis, in order: one thread per value of a row
template <typename T, int D>
__global__ __launch_bounds__(256) void diff_attn_join(DiffArgs a) {
  const int rows = a.N * a.G, per = 256 / (2 * D);
  const long long all = (long long)a.B * a.Hk * rows, row = (long long)blockIdx.x * per + threadIdx.x / (2 * D);
  if (row >= all) return;
  const int ch = threadIdx.x % (2 * D);
  float m0 = -INFINITY, m1 = -INFINITY;
  for (int s = 0; s < a.splits; ++s) {
    const float4 e = *(const float4*)(a.part_ml + (s * all + row) * 4);
    m0 = fmaxf(m0, e.x);
    m1 = fmaxf(m1, e.z);
  }
  float l0 = 0.f, l1 = 0.f, o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float4 e = *(const float4*)(a.part_ml + (s * all + row) * 4);
    const float* p = a.part_o + (s * all + row) * 4 * D + ch;
    const float w0 = e.x == -INFINITY ? 0.f : exp2f(e.x - m0), w1 = e.z == -INFINITY ? 0.f : exp2f(e.z - m1);
    l0 = fmaf(w0, e.y, l0);
    l1 = fmaf(w1, e.w, l1);
    o0 = fmaf(w0, p[0], o0);
    o1 = fmaf(w1, p[2 * D], o1);
  }
  const int bh = (int)(row / rows), r = (int)(row % rows), b = bh / a.Hk, head = bh % a.Hk * a.G + r % a.G, n = r / a.G;
  o0 *= l0 > 0.f ? 1.f / l0 : l0;
  o1 *= l1 > 0.f ? 1.f / l1 : l1;
  const long long at = ((long long)b * a.N + n) * a.H + head;
  ((T*)a.out)[at * 2 * D + ch] = (T)(o0 - lam_of<T>(a, head) * o1);
  if (a.o12) {
    a.o12[at * 4 * D + ch] = o0;
    a.o12[at * 4 * D + 2 * D + ch] = o1;
  }
  if (a.lse && ch == 0) {
    float* e = a.lse + ((long long)b * a.H + head) * 2 * a.N + n;
    e[0] = l0 == 0.f ? INFINITY : m0 + log2f(l0);
    e[a.N] = l1 == 0.f ? INFINITY : m1 + log2f(l1);
  }
}

// --------------------------------------------------------------------------------------------------------------- backward
// With G = dout v^T and delta_i = dout . o_i:  dS1 = A1 (G - delta1), dS2 = -lam A2 (G - delta2), dq_i = scale dS_i k_i, dk_i = scale dS_i^T q_i,
// dv = (A1 - lam A2)^T dout, dlam = -sum A2 G.  A and G are formed again from q, k, v, dout and the saved log sums, twice: once by rows (dq, delta,
// dlam) and once by keys (dk, dv), 14 instead of 10 products of N M D, so that no two workgroups add to one value and gradients do not depend on scheduling.
template <typename T, int D> struct BwdShape { static constexpr int KT = 32; };

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 1) void diff_attn_dq(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  constexpr int KT = BwdShape<T, D>::KT, NK = D / 16, NV = 2 * D / 16, NC = D / 32;
  constexpr unsigned long long kAll = (1ull << KT) - 1;
  __shared__ __attribute__((aligned(16))) char kt[2][KT * TL::kRow];
  __shared__ __attribute__((aligned(16))) char vt[2][KT * TL::kRow];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int rows = a.N * a.G, tiles = (rows + NW * 32 - 1) / (NW * 32);
  const unsigned id = by_xcd(blockIdx.x, gridDim.x);
  const int tile = tiles - 1 - (int)(id % tiles);
  const int bh = id / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int len = a.M;
  const int r0 = (tile * NW + wave) * 32, r = r0 + (lane & 31), rc = min(r, rows - 1);
  const int n = rc / a.G, head = hk * a.G + rc % a.G;
  const int off = len - a.N;
  const int lim = r >= rows ? -1 : a.causal ? min(n + off, len - 1) : len - 1;
  const int lim_lo = r0 + 31 >= rows ? -1 : a.causal ? min(r0 / a.G + off, len - 1) : len - 1;
  const int lim_hi = r0 >= rows ? -1 : a.causal ? min(min(r0 + 31, rows - 1) / a.G + off, len - 1) : len - 1;
  const int wg_hi = a.causal ? min(min((tile + 1) * NW * 32 - 1, rows - 1) / a.G + off, len - 1) : len - 1;
  const int t1 = max((wg_hi + KT) / KT, 0);
  const long long at = ((long long)b * a.N + n) * a.H + head;

  const T* q = (const T*)a.q + b * a.q_sb + n * a.q_sn + head * a.q_sh + 8 * h;
  const T* go = (const T*)a.dout + at * 2 * D + 8 * h;
  F qf[2][NK], gf[NV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[m][s] = load8<T>(q + m * a.q_sm + 16 * s);
#pragma unroll
  for (int s = 0; s < NV; ++s) gf[s] = load8<T>(go + 16 * s);
  float delta[2] = {0.f, 0.f}, lse[2];
  const long long st = ((long long)b * a.H + head) * 2 * a.N + n;
  {
    const float* oo = a.o12 + at * 4 * D + 8 * h;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int s = 0; s < NV; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) delta[m] = fmaf((float)gf[s][j], oo[m * 2 * D + 16 * s + j], delta[m]);
      delta[m] += __shfl_xor(delta[m], 32, 64);
      lse[m] = a.lse[st + m * a.N];
      if (h == 0 && r < rows) a.delta[st + m * a.N] = delta[m];
    }
  }
  const float lam = lam_of<T>(a, head);
  const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
  const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  f32x16 dq[2][NC];
  float dlam = 0.f;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) dq[m][c] = zero16();
  const typename TL::template Loader<KT, NW> lk(a.k_sn, a.k_sm, threadIdx.x), lv(a.v_sn, D, threadIdx.x);
  auto fetch = [&](int t, int buf) {
    lk(kt[buf], k + (long long)t * KT * a.k_sn, len - t * KT, threadIdx.x, wave);
    lv(vt[buf], v + (long long)t * KT * a.v_sn, len - t * KT, threadIdx.x, wave);
  };
  if (t1 > 0) fetch(0, 0);
  for (int t = 0; t < t1; ++t) {
    const int cur = t & 1, k0 = t * KT;
    unsigned long long seen = kAll;
    if (mask || k0 + KT > len) seen = keys_seen<KT>(mask, k0, len, lane);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1, cur ^ 1);
    if (seen == 0) continue;
    if (seen != kAll) {
      TL::template clear<KT, NW * 64>(kt[cur], seen, threadIdx.x);
      TL::template clear<KT, NW * 64>(vt[cur], seen, threadIdx.x);
      __syncthreads();
    }
    if (lim_hi < k0) continue;
    f32x16 s[2], g = zero16();
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s[m] = zero16();
#pragma unroll
      for (int i = 0; i < NK; ++i) s[m] = mma(TL::row(kt[cur], lane & 31, m * D + 16 * i + 8 * h), qf[m][i], s[m]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) g = mma(TL::row(vt[cur], lane & 31, 16 * i + 8 * h), gf[i], g);
    const bool part = (unsigned)seen != ~0u || k0 + 31 > lim_lo;
    const unsigned ok = part ? keys_of_lane((unsigned)seen, lim - k0, h) : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.c, -lse[0])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][i], a.c, -lse[1]));
      if (part) {
        p0 = (ok >> row_of(i, 0)) & 1 ? p0 : 0.f;
        p1 = (ok >> row_of(i, 0)) & 1 ? p1 : 0.f;
      }
      dlam = fmaf(p1, g[i], dlam);
      s[0][i] = p0 * (g[i] - delta[0]);
      s[1][i] = p1 * (g[i] - delta[1]) * -lam;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const F ds = pack<T>(s[m], i);
#pragma unroll
        for (int c = 0; c < NC; ++c) dq[m][c] = mma(TL::col(kt[cur], 16 * i, m * D + 32 * c, lane), ds, dq[m][c]);
      }
  }
  dlam += __shfl_xor(dlam, 32, 64);
  if (r >= rows) return;
  if (a.dq) {
    T* out = (T*)a.dq + at * 2 * D + 4 * h;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<T>(out + m * D + 32 * c + 8 * g, dq[m][c][4 * g] * a.scale, dq[m][c][4 * g + 1] * a.scale, dq[m][c][4 * g + 2] * a.scale, dq[m][c][4 * g + 3] * a.scale);
  }
  if (h == 0) a.dlam_rows[((long long)b * a.H + head) * a.N + n] = dlam;
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 1) void diff_attn_dkv(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  constexpr int QT = BwdShape<T, D>::KT, NK = D / 16, NV = 2 * D / 16, NC = D / 32, ND = 2 * D / 32;
  __shared__ __attribute__((aligned(16))) char qt[2][QT * TL::kRow];
  __shared__ __attribute__((aligned(16))) char gt[2][QT * TL::kRow];
  __shared__ __attribute__((aligned(16))) float stat[2][4][QT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int tiles = (a.M + NW * 32 - 1) / (NW * 32);
  const unsigned id = by_xcd(blockIdx.x, gridDim.x);
  const int tile = (int)(id % tiles), bh = id / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int off = a.M - a.N;
  const int k0 = (tile * NW + wave) * 32, key = k0 + (lane & 31), kc = min(key, a.M - 1);
  const T* k = (const T*)a.k + b * a.k_sb + kc * a.k_sn + hk * a.k_sh + 8 * h;
  const T* v = (const T*)a.v + b * a.v_sb + kc * a.v_sn + hk * a.v_sh + 8 * h;
  const bool seen = key < a.M && (!a.mask || a.mask[b * a.mask_sb + kc]);
  F kf[2][NK], vf[NV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) kf[m][s] = load8<T>(k + m * a.k_sm + 16 * s);
#pragma unroll
  for (int s = 0; s < NV; ++s) vf[s] = load8<T>(v + 16 * s);
  f32x16 dk[2][NC], dv[ND];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) dk[m][c] = zero16();
#pragma unroll
  for (int c = 0; c < ND; ++c) dv[c] = zero16();

  // queries that see the workgroup's first key, in tiles, of each head that shares it
  const int first = a.causal ? max(0, tile * NW * 32 - off) / QT : 0, nq = (a.N + QT - 1) / QT - first, total = max(nq, 0) * a.G;
  const typename TL::template Loader<QT, NW> lq(a.q_sn, a.q_sm, threadIdx.x), lg((long long)a.H * 2 * D, D, threadIdx.x);
  auto fetch = [&](int i, int buf) {
    const int head = hk * a.G + i / nq, n0 = (first + i % nq) * QT;
    lq(qt[buf], (const T*)a.q + b * a.q_sb + head * a.q_sh + n0 * a.q_sn, a.N - n0, threadIdx.x, wave);
    lg(gt[buf], (const T*)a.dout + (((long long)b * a.N + n0) * a.H + head) * 2 * D, a.N - n0, threadIdx.x, wave);
    const long long st = ((long long)b * a.H + head) * 2 * a.N;
    for (int w = wave; w < 2; w += NW) {                                        // lse of both maps, then delta of both: 32 values each
      const float* src = (w == 0 ? a.lse : a.delta) + st + (long long)h * a.N + min(n0 + (lane & 31), a.N - 1);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)(&stat[buf][2 * w][0]), 4, 0, 0);
    }
  };
  if (total > 0) fetch(0, 0);
  for (int i = 0; i < total; ++i) {
    const int cur = i & 1, n0 = (first + i % nq) * QT;
    const float lam = lam_of<T>(a, hk * a.G + i / nq);
    __syncthreads();
    if (i + 1 < total) fetch(i + 1, cur ^ 1);
    if (a.causal && n0 + QT - 1 + off < k0) continue;                           // (this wave's keys lie behind all of them)
    f32x16 s[2], g = zero16();
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s[m] = zero16();
#pragma unroll
      for (int j = 0; j < NK; ++j) s[m] = mma(TL::row(qt[cur], lane & 31, m * D + 16 * j + 8 * h), kf[m][j], s[m]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) g = mma(TL::row(gt[cur], lane & 31, 16 * j + 8 * h), vf[j], g);
    const bool part = n0 + QT > a.N || (a.causal && k0 + 31 > n0 + off);
    f32x16 pc;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 e0 = *(const float4*)&stat[cur][0][8 * u + 4 * h], e1 = *(const float4*)&stat[cur][1][8 * u + 4 * h];
      const float4 d0 = *(const float4*)&stat[cur][2][8 * u + 4 * h], d1 = *(const float4*)&stat[cur][3][8 * u + 4 * h];
      const float E0[4] = {e0.x, e0.y, e0.z, e0.w}, E1[4] = {e1.x, e1.y, e1.z, e1.w}, D0[4] = {d0.x, d0.y, d0.z, d0.w}, D1[4] = {d1.x, d1.y, d1.z, d1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = 4 * u + j;
        float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][x], a.c, -E0[j])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][x], a.c, -E1[j]));
        if (part) {
          const int n = n0 + 8 * u + 4 * h + j;
          const bool ok = n < a.N && (!a.causal || key <= n + off);
          p0 = ok ? p0 : 0.f;
          p1 = ok ? p1 : 0.f;
        }
        pc[x] = fmaf(-lam, p1, p0);
        s[0][x] = p0 * (g[x] - D0[j]);
        s[1][x] = p1 * (g[x] - D1[j]) * -lam;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const F p = pack<T>(pc, j);
#pragma unroll
      for (int c = 0; c < ND; ++c) dv[c] = mma(TL::col(gt[cur], 16 * j, 32 * c, lane), p, dv[c]);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const F ds = pack<T>(s[m], j);
#pragma unroll
        for (int c = 0; c < NC; ++c) dk[m][c] = mma(TL::col(qt[cur], 16 * j, m * D + 32 * c, lane), ds, dk[m][c]);
      }
    }
  }
  if (key >= a.M) return;
  // (a key nobody sees has gradient 0; what its lanes hold came of values that may be anything, and stayed in their own columns)
  const long long at = (((long long)b * a.M + key) * a.Hk + hk) * 2 * D + 4 * h;
#pragma unroll
  for (int c = 0; c < ND; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4<T>((T*)a.dv + at + 32 * c + 8 * g, seen ? dv[c][4 * g] : 0.f, seen ? dv[c][4 * g + 1] : 0.f, seen ? dv[c][4 * g + 2] : 0.f, seen ? dv[c][4 * g + 3] : 0.f);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4<T>((T*)a.dk + at + m * D + 32 * c + 8 * g, seen ? dk[m][c][4 * g] * a.scale : 0.f, seen ? dk[m][c][4 * g + 1] * a.scale : 0.f,
                  seen ? dk[m][c][4 * g + 2] * a.scale : 0.f, seen ? dk[m][c][4 * g + 3] * a.scale : 0.f);
}

// dlam[h] = - the sum of its rows' shares, in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void diff_attn_dlam(DiffArgs a) {
  __shared__ float s[16];
  const int head = blockIdx.x;
  float v = 0.f;
  for (int i = threadIdx.x; i < a.B * a.N; i += 1024) v += a.dlam_rows[((long long)(i / a.N) * a.H + head) * a.N + i % a.N];
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float w = 0.f;
    for (int i = 0; i < 16; ++i) w += s[i];
    if (a.lam_f32) ((float*)a.dlam)[head] = -w;
    else ((T*)a.dlam)[head] = (T)-w;
  }
}

}  // namespace tok
}  // namespace pgrf
