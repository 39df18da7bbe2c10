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

__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)(const char*)p; }

__device__ __forceinline__ const void* same_in_all_lanes(const void* p) {
  const unsigned long long v = (unsigned long long)p;
  return (const void*)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// 16 (or 4) bytes of every lane, from base + its offset, straight into LDS, one lane behind the other from the wave's address `to`.  As assembly, because the compiler lets a
// transposed read wait for every such load in flight, though it goes to another tile.  Nothing but landed() waits for these.  Nor does the compiler keep the distances inside
// assembly that the chip asks for: five wait states from a vector instruction that writes a scalar register (the base comes from readfirstlane) to the instruction on memory that
// reads it, one from a write of m0.  The five stand in front of every load (tests/test_token_isa.py looks them over in the built code).
__device__ __forceinline__ void fetch16(const void* base, unsigned off, unsigned to) {
  base = same_in_all_lanes(base);
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(to), "v"(off), "s"(base) : "memory");
}
// Four of them, to addresses `step` apart, behind one wait
template <int step>
__device__ __forceinline__ void fetch16x4(const void* base, const unsigned (&off)[4], unsigned to) {
  base = same_in_all_lanes(base);
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile(
      "s_nop 4\n\tglobal_load_lds_dwordx4 %2, %6\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %6\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %6\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %6"
      : "={m0}"(to)
      : "0"(to), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "i"(step)
      : "memory", "scc");
}
__device__ __forceinline__ void fetch4(const void* base, unsigned off, unsigned to) {
  base = same_in_all_lanes(base);
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(to), "v"(off), "s"(base) : "memory");
}
// What the wave fetched so far is in LDS.  Every kernel ends behind one of these, whatever its loops skipped: a workgroup's LDS may not go to another with loads on their way.
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Everything that the workgroup's waves fetched so far is in LDS, and their reads so far are done
__device__ __forceinline__ void fetched() {
  landed();
  __syncthreads();
}

// A tile of rows of 2 D values in LDS (at a multiple of 256 bytes), in chunks of 16 bytes; chunk c of row r lies at place c ^ turn(r).  turn swaps bits of the row
// number so that the lanes that LDS serves at a time (256 bytes: 64 banks) meet every bank once, both where 16 rows hand out the same chunk and where the transposed
// reads take 64 bytes of 4 rows (16 bits), or 128 of 2 (float).  (b128 reads of 16 rows: 4.3 cycles; with 8 different places 8.4, with the plain layout 64.)
template <typename T, int D>
struct Tile {
  static constexpr int kRow = 2 * D * (int)sizeof(T), kChunks = kRow / 16, kPer = 16 / (int)sizeof(T);
  using F = typename Frag8<T>::type;
  static __host__ __device__ constexpr int turn(int r) {
    return kChunks == 8      ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3)
           : sizeof(T) == 2  ? (r & 3) << 2 | ((r >> 2) & 3)
                             : ((r >> 2) & 1) << 3 | ((r >> 3) & 1) << 2 | (r & 3);
  }
  // Where a lane reads: turn is a swap of bits, so every place a lane needs is one of these two with some constant bits flipped, and a constant behind
  struct Lane {
    unsigned row, col;
    __device__ explicit Lane(int lane) {
      const int r = lane & 31, h = lane >> 5;
      if constexpr (sizeof(T) == 2) {
        row = r * kRow + ((h ^ turn(r)) << 4);
        // ds_read_b64_tr: the 16 lanes of a group hand in 4 rows x 16 values (4 values each) and each gets a column of 4
        const int i = lane & 15, rr = 4 * h + (i >> 2), c = ((lane & 16) >> 3) + ((i & 3) >> 1);
        col = rr * kRow + ((c ^ turn(rr)) << 4) + (i & 1) * 8;
      } else {
        row = r * kRow + (((2 * h) ^ turn(r)) << 4);
        col = 4 * h * kRow + (((r >> 2) ^ turn(4 * h)) << 4) + (r & 3) * 4;
      }
    }
  };
  static constexpr int kLow = kChunks < 16 ? kChunks : 16;                     // chunks that turn moves among themselves
  template <typename W>
  static __device__ __forceinline__ W read(unsigned at) { return *(__attribute__((address_space(3))) W*)(size_t)at; }
  static __device__ __forceinline__ unsigned lds(const char* t) { return lds_address(t); }

  // 8 values, 16 q + 8 h .. + 7, of row `lane & 31`
  static __device__ __forceinline__ F row(const char* t, const Lane& l, int q) {
    const unsigned b = lds(t) + l.row;
    if constexpr (sizeof(T) == 2) {
      return read<F>((b ^ (2 * q % kLow << 4)) + 2 * q / kLow * kLow * 16);
    } else {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const int c = 4 * q;
      const f4 lo = read<f4>((b ^ (c % kLow << 4)) + c / kLow * kLow * 16), hi = read<f4>((b ^ ((c + 1) % kLow << 4)) + c / kLow * kLow * 16);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // the transposed fragment: value 32 c + (lane & 31) of rows 16 s + 4 h + {0..3, 8..11}
  static __device__ __forceinline__ F col(const char* t, const Lane& l, int s, int c) {
    const unsigned b = lds(t) + l.col;
    if constexpr (sizeof(T) == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const int k = 4 * c, behind = s * 16 * kRow + k / kLow * kLow * 16;
      const unsigned p = (b ^ (k % kLow << 4)) + behind, q = (b ^ ((k % kLow ^ turn(8)) << 4)) + behind + 8 * kRow;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(size_t)p);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(size_t)q);
      const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(F, v);
    } else {
      F v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = (j & 3) + 8 * (j >> 2), k = 8 * c;
        v[j] = read<float>((b ^ ((k % kLow ^ turn(r)) << 4)) + (16 * s + r) * kRow + k / kLow * kLow * 16);
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
    int row0, chunk, sn, sm;
    __device__ Loader(long long sn_, long long sm_, int tid) : row0(tid / kChunks), chunk((tid % kChunks) ^ turn(tid / kChunks)), sn((int)sn_), sm((int)sm_) {}
    __device__ __forceinline__ int val(int i) const {
      const int e = (chunk ^ turn(i * kRowsPer)) * kPer;                       // (row0 < kRowsPer, a power of two: the bits of the two stay apart)
      return e >= D ? e - D + sm : e;
    }
    // base: the tile's first row; rows from `rows` on repeat the last one, rows below `from` that one (they are masked)
    __device__ __forceinline__ void operator()(char* t, const T* base, int rows, int tid, int wave, int from = -0x7fffffff - 1) const {
      unsigned off[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int r = row0 + i * kRowsPer, g = max(min(r, rows - 1), from);
        off[i] = (g * sn + val(i)) * (int)sizeof(T);
      }
      if constexpr (kSteps % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kSteps; i += 4) fetch16x4<NW * 1024>(base, *(const unsigned(*)[4])(off + i), lds(t) + (i * NW + wave) * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) fetch16(base, off[i], lds(t) + (i * NW + wave) * 1024);
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
  // bf16, where products bound the forward pass: v in f16 [B*Hk][M][2D] times 2^v_exp of the key head (kWide: not), and what v_exp comes from, in parts of the keys
  void* v16;
  int* v_exp;                     // [B*Hk]
  float* v_sizes;                 // [B*Hk][v_parts][2]: the largest |v|, and the smallest among the keys' largest
  int v_parts;
  // a key axis cut into `splits`: partial [splits][B*Hk][N*G] rows of 2 x 2D values and (m1, l1, m2, l2)
  int splits;
  float *part_o, *part_ml;
  // backward
  const void* dout;               // [B,N,H,2D] contiguous
  float* delta;                   // [B,H,2,N]: dout . o_i
  float* dlam_part;               // [B*Hk][units][G]: parts of -dlam, by wave of the dq kernel (G a power of two up to 32) or by token, of every share
  float* sizes;                   // f16: [B*Hk][size_parts][2], the largest |v_j|^2 and |dout_i|^2 of a part of the key head's keys and rows
  int size_parts;
  void *dq, *dk, *dv, *dlam;
  // a workgroup's blocks cut into shares: partial gradients [shares][...] in float
  int q_shares, kv_shares;
  float *dq_part, *dk_part, *dv_part;
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

// Products 0 .. N - 1 in this order, the fragment of each read AHEAD products before it, and a share of other work behind each.  Left to itself the compiler reads
// each fragment right before its product, waits for it, and puts the other work behind all of them; the fences keep it to this order.
template <typename F, int N, int AHEAD, class Read, class Product, class Work>
__device__ __forceinline__ void weave(Read read, Product product, Work work) {
  F f[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) f[(i + AHEAD) % (AHEAD + 1)] = read(i + AHEAD);
    product(i, f[i % (AHEAD + 1)]);
    work(i);
    __builtin_amdgcn_sched_barrier(0);
  }
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
// How probabilities go into the product with v (16 bits).  kOne: rounded to the tensors' type.  What the two maps have in common cancels in out and their roundings do not: of
// independent maps out is off by 0.0026 of its norm in bf16, where 0.0017 is its own rounding, of sharp maps that nearly cancel by
// 0.0068 (scores of 3, nearly equal, 0.9 of the second taken off; 0.0018 in f16).
// kTwo: in two pieces, what the type holds and what that leaves: nothing is lost, for 20 products of N M D in place of 12.  Taken where memory bounds the kernel: up to 32 rows
// (caches as in cut_fwd: 246 us both ways), and up to 64 keys (2048 rays of 64 samples, 4 heads x 64, bf16: 164 us in one piece, 166 in two; x 32: 50, 52; 1024 rows
// on 64 keys, 64 x 8 heads x 32: 40, 45; x 128: 268, 283).
// kInF16 (bf16): v goes to f16 first, by a power of two that is exact but for values 2^-13 of their own key's largest, and with it the probabilities, which have 8 times
// finer steps there at the same rate.  That is two launches over v, and one for key heads whose keys differ too much for f16's range (kWide), which take kTwo: 6 + 7 + 5 us for
// 8093 keys of 4 heads x 128.  Taken where products bound a long kernel (2 x 8192, 8 heads x 64, training: 2866 us in one piece, 2926 in f16, 3290 in two; 4001 of 8093, 16/4 heads
// x 128, causal: 615, 651, 870).  All other sizes, and f16 itself beyond 64 keys, keep kOne.
enum { kOne = 0, kTwo = 1, kInF16 = 2 };
constexpr int kWide = 1 << 20;

template <typename T, int D, int NW, int HOW> struct FwdShape {
  static_assert(D < 128 || NW > 1, "a pair of waves at D = 128");
  static constexpr int MPW = D == 128 ? 1 : 2, RW = NW * MPW / 2;              // RW: groups of 32 rows in the workgroup
  static constexpr int KT = 32;                                                // keys of a block
  // Float from D = 64 on: one wave on a SIMD (its operands take twice the registers) with three blocks in work.  All others: two waves on a SIMD, but for a workgroup of one
  // wave, which memory bounds (over caches 245 us with all registers it wants, 267 with half of them).
  static constexpr bool kWeave = sizeof(T) == 4 && D > 32;
  static constexpr int kMinWaves = kWeave || NW == 1 ? 1 : 2;
  static constexpr int kTileKeys = sizeof(T) == 2 && RW == 4 ? 64 : 32;        // keys between barriers: fewer barriers where LDS holds two such tiles
  static constexpr bool kTwoPieces = HOW == kTwo;
  using V = typename std::conditional<HOW == kInF16, f16, T>::type;            // v and the probabilities in their product
};

// Scores of a block: S^T of MPW maps
template <typename T, int D, int MPW>
__device__ __forceinline__ void scores(f32x16 (&s)[MPW], const char* kt, const typename Frag8<T>::type (&qf)[MPW][D / 16], int map0, const typename Tile<T, D>::Lane& at) {
#pragma unroll
  for (int m = 0; m < MPW; ++m) s[m] = zero16();
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int m = 0; m < MPW; ++m) s[m] = mma(Tile<T, D>::row(kt, at, (map0 + m) * (D / 16) + i), qf[m][i], s[m]);
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

// One pass over the keys in blocks of 32 with the running maximum and sum of each row's softmax.  What bounds it: per block and wave at D = 64 the matrix pipe has 24
// products of 32x32x16 (386 ns at its peak) and the vector pipe 96 FMAs and 32 exponentials with their sums and roundings (over 312 ns); side by side the two take 471 ns
// at best, and here they are busy for 45% and 57% of the time (2 x 8192 rows and keys, 8 heads, bf16: 820-855 us, 960-1000 TFLOP/s, as at D = 128, where no exponential is left over; the first calls on an idle card take 13% longer).  With kWeave a wave has three blocks in work: while block j goes through its exponentials, the matrix pipe
// forms the scores of block j + 1 and adds block j - 1 times its values, in one stretch of code without a branch; masks and a new maximum are dealt with in front of it.
template <typename T, int D, int NW, int HOW>
__global__ __launch_bounds__(NW * 64, (FwdShape<T, D, NW, HOW>::kMinWaves)) void diff_attn_fwd(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  using Sh = FwdShape<T, D, NW, HOW>;
  using VT = typename Sh::V;
  using TV = Tile<VT, D>;
  using FV = typename Frag8<VT>::type;
  constexpr int KT = Sh::KT, MPW = Sh::MPW, NK = D / 16, NC = 2 * D / 32, RW = Sh::RW;
  constexpr int kTile = KT * TL::kRow;
  constexpr int BT = Sh::kTileKeys / KT;                                         // blocks between barriers
  __shared__ __attribute__((aligned(1024))) char tiles_lds[4 * BT * kTile];        // two tiles of k, two of v
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const typename TL::Lane at(lane);
  const typename TV::Lane atv(lane);
  const int group = MPW == 2 ? wave : wave >> 1, map0 = MPW == 2 ? 0 : wave & 1;
  const int rows = a.N * a.G, tiles = (rows + RW * 32 - 1) / (RW * 32);
  // Workgroups side by side: the tiles of rows of one key head, on one XCD, so that they find its keys in its L2 (causal: the longest rows first).  Where there is one tile,
  // the key heads of the same keys, which stand side by side in memory, and no XCD gets more of the longer entries than another
  unsigned id = tiles == 1 ? blockIdx.x : by_xcd(blockIdx.x, gridDim.x);
  int split, tile, bh;
  if (tiles == 1) {
    const int heads = id % a.Hk;
    id /= a.Hk;
    split = id % a.splits;
    bh = id / a.splits * a.Hk + heads;
    tile = 0;
  } else {
    split = id % a.splits;
    id /= a.splits;
    tile = tiles - 1 - (int)(id % tiles);
    bh = id / tiles;
  }
  const int b = bh / a.Hk, hk = bh % a.Hk;
  if constexpr (HOW == kInF16) {
    if (a.v_exp[bh] == kWide) return;
  } else if constexpr (HOW == kTwo) {
    if (a.v_exp && a.v_exp[bh] != kWide) return;
  }
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.M) : a.M;
  const int r0 = (tile * RW + group) * 32, r = r0 + (lane & 31), rc = min(r, rows - 1);
  const int n = rc / a.G, head = hk * a.G + rc % a.G;
  // the last key a row sees, of the wave's first and last row, and of the workgroup's last row
  const int off = len - a.N;
  const int lim = r >= rows ? -1 : a.causal ? min(n + off, len - 1) : len - 1;
  const int lim_lo = r0 + 31 >= rows ? -1 : a.causal ? min(r0 / a.G + off, len - 1) : len - 1;
  const int lim_hi = r0 >= rows ? -1 : a.causal ? min(min(r0 + 31, rows - 1) / a.G + off, len - 1) : len - 1;
  const int wg_hi = a.causal ? min(min((tile + 1) * RW * 32 - 1, rows - 1) / a.G + off, len - 1) : len - 1;
  // a share is the same number of tiles for every entry, so that long entries have more of them and not longer ones
  const int all = (wg_hi + KT * BT) / (KT * BT), per = ((a.M + KT * BT - 1) / (KT * BT) + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(all, t0 + per);                         // tiles

  const T* q = (const T*)a.q + b * a.q_sb + n * a.q_sn + head * a.q_sh + map0 * a.q_sm + 8 * h;
  F qf[MPW][NK];
#pragma unroll
  for (int m = 0; m < MPW; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[m][s] = load8<T>(q + m * a.q_sm + 16 * s);

  const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
  const VT* v = HOW == kInF16 ? (const VT*)a.v16 + (long long)bh * a.M * 2 * D : (const VT*)a.v + b * a.v_sb + hk * a.v_sh;
  const long long v_sn = HOW == kInF16 ? 2 * D : a.v_sn;
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const typename TL::template Loader<KT, NW> lk(a.k_sn, a.k_sm, tid);
  const typename TV::template Loader<KT, NW> lv(v_sn, D, tid);
  auto ktile = [&](int t) { return tiles_lds + (t & 1) * kTile; };
  auto vtile = [&](int t) { return tiles_lds + 2 * kTile + (t & 1) * kTile; };
  auto fetch_k = [&](int t) { lk(ktile(t), k + (long long)t * KT * a.k_sn, len - t * KT, tid, wave); };
  auto fetch_v = [&](int t) { lv(vtile(t), v + (long long)t * KT * v_sn, len - t * KT, tid, wave); };

  f32x16 o[MPW][NC], s[MPW];
  FV p[MPW][2], rest[Sh::kTwoPieces ? MPW : 1][2];
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
      for (int j = 0; j < 8; ++j) p[m][i][j] = (VT)0.f;
  }
  auto add_block = [&](const char* vt) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const FV vf = TV::col(vt, atv, i, c);
#pragma unroll
        for (int m = 0; m < MPW; ++m) o[m][c] = mma(vf, p[m][i], o[m][c]);
      }
  };

  auto hide = [&](unsigned seen, int k0) {                                      // masked keys of a block
    if (seen != ~0u || k0 + 31 > lim_lo) {
      const unsigned ok = keys_of_lane(seen, lim - k0, h);
#pragma unroll
      for (int m = 0; m < MPW; ++m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[m][i] = (ok >> row_of(i, 0)) & 1 ? s[m][i] : -INFINITY;
        top[m] = top_of(s[m]);
      }
    }
  };
  // The running maximum follows only where a row outgrew it by 2^8, and by a whole power of two: sums and values stay in range, and what was rounded before
  // scales without another rounding
  auto grow = [&]() {
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
      const float up = with_other_half(top[m]) * a.c;
      if (__any(up > mx[m] + 8.f)) {
        const float more = fmaxf(ceilf(up - mx[m]), 0.f), f = mx[m] == -INFINITY ? 1.f : ldexpf(1.f, -(int)fminf(more, 1000.f));
        mx[m] = mx[m] == -INFINITY ? up : mx[m] + more;
        l[m] *= f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[m][c] *= f;
        if constexpr (Sh::kWeave)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[m][i][j] = (VT)((float)p[m][i][j] * f);
      }
    }
  };
  if constexpr (Sh::kWeave) {
    if (t0 < t1) {
      fetch_k(t0);
      for (int i = tid; i < kTile / 16; i += NW * 64) *(float4*)(vtile(t0 - 1) + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);   // (its probabilities are 0)
      unsigned seen = ~0u;
      fetched();
      if (t0 + 1 < t1) fetch_k(t0 + 1);
      scores<T, D, MPW>(s, ktile(t0), qf, map0, at);
#pragma unroll
      for (int m = 0; m < MPW; ++m) top[m] = top_of(s[m]);
      for (int t = t0; t < t1; ++t) {
        const int k0 = t * KT;
        const unsigned before = seen;
        seen = ~0u;
        if (mask || k0 + KT > len) seen = (unsigned)keys_seen<KT>(mask, k0, len, lane);
        fetched();                                                         // k of t + 1 and v of t - 1 have come; nobody reads k of t or v of t - 2 any more
        if (t + 2 < t1) fetch_k(t + 2);
        if (before != ~0u) {                                                     // what stands in masked values may be anything, and 0 * NaN is NaN
          TL::template clear<KT, NW * 64>(vtile(t - 1), before, tid);
          __syncthreads();
        }
        fetch_v(t);
        hide(seen, k0);
        grow();
        f32x16 next[MPW];
        const char *kn = ktile(t + 1), *vb = vtile(t - 1);                       // (behind the last block: scores of whatever stands there, unused)
        float base[MPW], sum[MPW];
        F pn[MPW][2];
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
          next[m] = zero16();
          base[m] = mx[m] == -INFINITY ? 0.f : mx[m];
          sum[m] = 0.f;
        }
        constexpr int NS = NK * MPW, NA = 2 * NC, NP = NS + NA;                   // fragments of k, of v; every one of v serves MPW products
        weave<F, NP, 3>(
            [&](int i) {
              return i < NS ? TL::row(kn, at, (map0 + i % MPW) * NK + i / MPW) : TL::col(vb, at, (i - NS) / NC, (i - NS) % NC);
            },
            [&](int i, const F& f) {
              if (i < NS) {
                next[i % MPW] = mma(f, qf[i % MPW][i / MPW], next[i % MPW]);
              } else {
                const int c = (i - NS) % NC;
#pragma unroll
                for (int m = 0; m < MPW; ++m) o[m][c] = mma(f, p[m][(i - NS) / NC], o[m][c]);
              }
            },
            [&](int i) {
#pragma unroll
              for (int x = 16 * MPW * i / NP; x < 16 * MPW * (i + 1) / NP; ++x) {
                const int m = x / 16, e = x % 16;
                const float w = __builtin_amdgcn_exp2f(fmaf(s[m][e], a.c, -base[m]));
                sum[m] += w;
                pn[m][e / 8][e % 8] = (T)w;
              }
            });
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
          l[m] += sum[m];
          p[m][0] = pn[m][0];
          p[m][1] = pn[m][1];
          s[m] = next[m];
          top[m] = top_of(s[m]);
        }
      }
      fetched();
      if (seen != ~0u) {
        TL::template clear<KT, NW * 64>(vtile(t1 - 1), seen, tid);
        __syncthreads();
      }
      add_block(vtile(t1 - 1));
    }
  } else if (t0 < t1) {
    // two or more waves on a SIMD: one's exponentials run beside another's products, block by block
    constexpr int kB = BT * KT;
    const typename TL::template Loader<kB, NW> bk(a.k_sn, a.k_sm, tid);
    const typename TV::template Loader<kB, NW> bv(v_sn, D, tid);
    auto tile_at = [&](int t) { return tiles_lds + (t & 1) * 2 * BT * kTile; };  // k, then v
    auto fetch = [&](int t) {
      bk(tile_at(t), k + (long long)t * kB * a.k_sn, len - t * kB, tid, wave);
      bv(tile_at(t) + BT * kTile, v + (long long)t * kB * v_sn, len - t * kB, tid, wave);
    };
    fetch(t0);
    for (int t = t0; t < t1; ++t) {
      const char *kt = tile_at(t), *vt = kt + BT * kTile;
      unsigned long long seen = kB == 64 ? ~0ull : 0xffffffffull;
      if (mask || t * kB + kB > len) seen = keys_seen<kB>(mask, t * kB, len, lane);
      fetched();                                                         // tile t has come; nobody reads the other any more
      if (t + 1 < t1) fetch(t + 1);
      if (seen == 0) continue;
      if (seen != (kB == 64 ? ~0ull : 0xffffffffull)) {
        TL::template clear<kB, NW * 64>((char*)vt, seen, tid);
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < BT; ++u) {
        const int k0 = (t * BT + u) * KT;
        if (k0 > lim_hi) break;
        const char *kb = kt + u * kTile, *vb = vt + u * kTile;
#pragma unroll
        for (int m = 0; m < MPW; ++m) s[m] = zero16();
        weave<F, NK * MPW, 2>([&](int i) { return TL::row(kb, at, (map0 + i % MPW) * NK + i / MPW); },
                              [&](int i, const F& f) { s[i % MPW] = mma(f, qf[i % MPW][i / MPW], s[i % MPW]); }, [](int) {});
#pragma unroll
        for (int m = 0; m < MPW; ++m) top[m] = top_of(s[m]);
        hide((unsigned)(seen >> (KT * u)), k0);
        grow();
#pragma unroll
        for (int m = 0; m < MPW; ++m) {
          const float base = mx[m] == -INFINITY ? 0.f : mx[m];
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float w = __builtin_amdgcn_exp2f(fmaf(s[m][e], a.c, -base));
            sum += w;
            p[m][e / 8][e % 8] = (VT)w;
            if constexpr (Sh::kTwoPieces) rest[m][e / 8][e % 8] = (VT)(w - (float)(VT)w);
          }
          l[m] += sum;
        }
        weave<FV, 2 * NC, 2>([&](int i) { return TV::col(vb, atv, i / NC, i % NC); },
                            [&](int i, const FV& f) {
#pragma unroll
                              for (int m = 0; m < MPW; ++m) {
                                o[m][i % NC] = mma(f, p[m][i / NC], o[m][i % NC]);
                                if constexpr (Sh::kTwoPieces) o[m][i % NC] = mma(f, rest[m][i / NC], o[m][i % NC]);
                              }
                            },
                            [](int) {});
      }
    }
  }
  landed();
#pragma unroll
  for (int m = 0; m < MPW; ++m) l[m] += __shfl_xor(l[m], 32, 64);
  if constexpr (HOW == kInF16) {
    const float undo = ldexpf(1.f, -a.v_exp[bh]);
#pragma unroll
    for (int m = 0; m < MPW; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c) o[m][c] *= undo;
  }
  const bool live = r < rows;
  if (a.splits > 1) {
    if (!live) return;
    if (t0 >= t1) {                                                            // (an empty share: only its sums are read)
      if (h == 0)
#pragma unroll
        for (int m = 0; m < MPW; ++m) *(float2*)(a.part_ml + (((long long)split * a.B * a.Hk + bh) * rows + r) * 4 + 2 * (map0 + m)) = make_float2(-INFINITY, 0.f);
      return;
    }
    const long long pat = ((long long)split * a.B * a.Hk + bh) * rows + r;
    float* po = a.part_o + pat * 4 * D + map0 * 2 * D + 4 * h;
#pragma unroll
    for (int m = 0; m < MPW; ++m) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<float>(po + m * 2 * D + 32 * c + 8 * g, o[m][c][4 * g], o[m][c][4 * g + 1], o[m][c][4 * g + 2], o[m][c][4 * g + 3]);
      if (h == 0) *(float2*)(a.part_ml + pat * 4 + 2 * (map0 + m)) = make_float2(mx[m], l[m]);
    }
    return;
  }
  const float lam = lam_of<T>(a, head);
  const long long oat = ((long long)b * a.N + n) * a.H + head;
#pragma unroll
  for (int m = 0; m < MPW; ++m) {
    const float inv = l[m] > 0.f ? 1.f / l[m] : l[m];                          // (a NaN stays one)
#pragma unroll
    for (int c = 0; c < NC; ++c) o[m][c] *= inv;
    if (a.o12 && live) {
      float* oo = a.o12 + oat * 4 * D + (map0 + m) * 2 * D + 4 * h;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) store4<float>(oo + 32 * c + 8 * g, o[m][c][4 * g], o[m][c][4 * g + 1], o[m][c][4 * g + 2], o[m][c][4 * g + 3]);
    }
    if (a.lse && live && h == 0) a.lse[(((long long)b * a.H + head) * 2 + map0 + m) * a.N + n] = l[m] == 0.f ? INFINITY : mx[m] + log2f(l[m]);
  }
  T* out = (T*)a.out + oat * 2 * D + 4 * h;
  if constexpr (MPW == 1) {
    // the second map's waves hand their values over through LDS, as many column blocks at a time as the tiles' room holds
    constexpr int kFit = 4 * BT * kTile / (RW * 64 * 64), kAt = kFit < NC ? kFit : NC;
    static_assert(kAt >= 1 && NC % kAt == 0, "");
    float* room = (float*)tiles_lds + group * kAt * 16 * 64 + lane;
    for (int c0 = 0; c0 < NC; c0 += kAt) {
      fetched();                                                         // (also: the tiles are read)
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

// The largest |v| of keys that are seen, and the smallest of their largest (finite values; keys of zeros aside), in parts
template <typename T, int D>
__global__ __launch_bounds__(256) void diff_attn_v_sizes(DiffArgs a) {
  using F = typename Frag8<T>::type;
  constexpr int L = 2 * D / 8, kRows = 256 / L;
  __shared__ float2 both[4];
  const int tid = threadIdx.x, part = blockIdx.x % a.v_parts, bh = blockIdx.x / a.v_parts, b = bh / a.Hk, hk = bh % a.Hk;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.M) : a.M;
  const int keys = (a.M + a.v_parts - 1) / a.v_parts, k1 = min(part * keys + keys, len);
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh + tid % L * 8;
  float most = 0.f, least = INFINITY;
  for (int k = part * keys + tid / L; k < k1; k += 4 * kRows) {
    F x[4];
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = min(k + j * kRows, k1 - 1);
      x[j] = load8<T>(v + at * a.v_sn);
      in[j] = !mask || mask[at];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = fabsf((float)x[j][i]);
        m = u < INFINITY ? fmaxf(m, u) : m;
      }
#pragma unroll
      for (int o = L / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      most = in[j] ? fmaxf(most, m) : most;
      least = in[j] && m > 0.f ? fminf(least, m) : least;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    most = fmaxf(most, __shfl_xor(most, o, 64));
    least = fminf(least, __shfl_xor(least, o, 64));
  }
  if ((tid & 63) == 0) both[tid >> 6] = make_float2(most, least);
  __syncthreads();
  if (tid == 0)
    *(float2*)(a.v_sizes + 2ll * blockIdx.x) = make_float2(fmaxf(fmaxf(both[0].x, both[1].x), fmaxf(both[2].x, both[3].x)),
                                                           fminf(fminf(both[0].y, both[1].y), fminf(both[2].y, both[3].y)));
}

// v in f16, with the key head's largest value at 2^14: what is 2^-28 of it still has all its bits, and a key whose largest is 2^-15 of it those down to 2^-13 of its own
template <typename T, int D>
__global__ __launch_bounds__(256) void diff_attn_v16(DiffArgs a) {
  using F = typename Frag8<T>::type;
  constexpr int L = 2 * D / 8, kRows = 256 / L;
  const int tid = threadIdx.x, lane = tid & 63, part = blockIdx.x % a.v_parts, bh = blockIdx.x / a.v_parts, b = bh / a.Hk, hk = bh % a.Hk;
  float most = 0.f, least = INFINITY;
  for (int i = lane; i < a.v_parts; i += 64) {
    const float2 x = *(const float2*)(a.v_sizes + ((long long)bh * a.v_parts + i) * 2);
    most = fmaxf(most, x.x);
    least = fminf(least, x.y);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    most = fmaxf(most, __shfl_xor(most, o, 64));
    least = fminf(least, __shfl_xor(least, o, 64));
  }
  const bool wide = most > 0.f && ilogbf(most) - ilogbf(least) > 15;
  const int e = most > 0.f ? min(14 - ilogbf(most), 120) : 0;
  if (part == 0 && tid == 0) a.v_exp[bh] = wide ? kWide : e;
  if (wide) return;
  const float f = ldexpf(1.f, e);
  const int keys = (a.M + a.v_parts - 1) / a.v_parts, k1 = min(part * keys + keys, a.M);
  const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh + tid % L * 8;
  f16* out = (f16*)a.v16 + (long long)bh * a.M * 2 * D + tid % L * 8;
  for (int k = part * keys + tid / L; k < k1; k += 4 * kRows) {
    F x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = load8<T>(v + min(k + j * kRows, k1 - 1) * a.v_sn);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Frag8<f16>::type y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (f16)((float)x[j][i] * f);
      if (k + j * kRows < k1) *(Frag8<f16>::type*)(out + (long long)(k + j * kRows) * 2 * D) = y;
    }
  }
}

// Joins the shares of a cut key axis: S groups of threads take every S-th share of a row, four at a time so that their loads are on their way together (one after the other
// 128 shares took 70 us), and the groups are joined in order; one thread per value and group.
template <typename T, int D, int S>
__global__ __launch_bounds__(S > 1 ? 2 * D * S : 256) void diff_attn_join(DiffArgs a) {
  constexpr int kRows = S > 1 ? 1 : 256 / (2 * D);                             // rows of a workgroup
  __shared__ __attribute__((aligned(16))) float sums[S > 1 ? S : 1][4];
  __shared__ float values[S > 1 ? S : 1][2][2 * D];
  const int rows = a.N * a.G, ch = threadIdx.x % (2 * D), group = S > 1 ? threadIdx.x / (2 * D) : 0;
  const long long all = (long long)a.B * a.Hk * rows, row = (long long)blockIdx.x * kRows + (S > 1 ? 0 : threadIdx.x / (2 * D));
  if (row >= all) return;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2] = {0.f, 0.f};
  // adds up to four parts of (m1, l1, m2, l2) and two values; one that saw no key (its values were never written) counts for nothing
  auto add = [&](const float4 (&e)[4], const float (&v)[4][2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float top = m[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, k ? e[j].z : e[j].x);
      const float f = m[k] == -INFINITY ? 0.f : exp2f(m[k] - top);
      l[k] *= f;
      o[k] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float mj = k ? e[j].z : e[j].x, lj = k ? e[j].w : e[j].y, w = mj == -INFINITY ? 0.f : exp2f(mj - top);
        const bool none = e[j].x == -INFINITY && e[j].z == -INFINITY && e[j].y == 0.f && e[j].w == 0.f;
        l[k] = fmaf(w, lj, l[k]);
        o[k] = none ? o[k] : fmaf(w, v[j][k], o[k]);
      }
      m[k] = top;
    }
  };
  const float4 nothing = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
  for (int s = group; s < a.splits; s += 4 * S) {
    float4 e[4];
    float v[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long at = min(s + j * S, a.splits - 1) * all + row;           // (behind the last: read again, not counted)
      const float* p = a.part_o + at * 4 * D + ch;
      e[j] = *(const float4*)(a.part_ml + at * 4);
      v[j][0] = p[0];
      v[j][1] = p[2 * D];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (s + j * S >= a.splits) e[j] = nothing;
    add(e, v);
  }
  if constexpr (S > 1) {
    if (ch == 0) *(float4*)sums[group] = make_float4(m[0], l[0], m[1], l[1]);
    values[group][0][ch] = o[0];
    values[group][1][ch] = o[1];
    __syncthreads();
    if (group) return;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = o[0] = o[1] = 0.f;
#pragma unroll
    for (int g = 0; g < S; g += 4) {
      float4 e[4];
      float v[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = *(const float4*)sums[g + j];
        v[j][0] = values[g + j][0][ch];
        v[j][1] = values[g + j][1][ch];
      }
      add(e, v);
    }
  }
  const int bh = (int)(row / rows), r = (int)(row % rows), b = bh / a.Hk, head = bh % a.Hk * a.G + r % a.G, n = r / a.G;
#pragma unroll
  for (int k = 0; k < 2; ++k) o[k] *= l[k] > 0.f ? 1.f / l[k] : l[k];
  const long long at = ((long long)b * a.N + n) * a.H + head;
  ((T*)a.out)[at * 2 * D + ch] = (T)(o[0] - lam_of<T>(a, head) * o[1]);
  if (a.o12) {
    a.o12[at * 4 * D + ch] = o[0];
    a.o12[at * 4 * D + 2 * D + ch] = o[1];
  }
  if (a.lse && ch == 0) {
    float* e = a.lse + ((long long)b * a.H + head) * 2 * a.N + n;
    e[0] = l[0] == 0.f ? INFINITY : m[0] + log2f(l[0]);
    e[a.N] = l[1] == 0.f ? INFINITY : m[1] + log2f(l[1]);
  }
}

// --------------------------------------------------------------------------------------------------------------- backward
// With G = dout v^T and delta_i = dout . o_i:  dS1 = A1 (G - delta1), dS2 = -lam A2 (G - delta2), dq_i = scale dS_i k_i, dk_i = scale dS_i^T q_i,
// dv = (A1 - lam A2)^T dout, dlam = -sum A2 G.  A and G are formed again from q, k, v, dout and the saved log sums, twice: once by rows (dq, delta,
// dlam) and once by keys (dk, dv), 14 instead of 10 products of N M D, so that no two workgroups add to one value and gradients do not depend on scheduling.
//
// Two waves or more share a SIMD and run beside each other, but for dq and dk at D = 128 in 16 bits, whose registers leave a SIMD one wave: those weave three blocks as the
// forward kernel does.  Float does neither, as its products take eight times as long and hide the rest by themselves.  Both pipes are bound as in the forward kernel (2 x 8192,
// 8 heads, bf16, D = 64: dq 850-885 us, dk and dv 1130-1180 us, both 930-970 TFLOP/s).
// In f16 the backward pass brings what it rounds into the type's range by powers of two that the float sums' last factor takes out again.  A score gradient a (G - delta) is a
// probability, about 1 / M, times what is often a mean loss' gradient: rounded as it is, it is lost below 2^-25 where dq and dk are well in range (8192 keys, dout of 1e-4: dq
// off by 7%), and is infinite above 65504.  |a (G - delta)| is at most 2 |dout_i| |v_j| and |a1 - lam a2| at most 1 + |lam|; with those at 2^14 what is 2^-28 of them still
// has all its bits.  dq sums over a row, so its factor is the row's; dk and dv sum over the rows of a key head, so theirs is the key head's.  bf16 has float's range.
template <typename T> constexpr bool kRanged = std::is_same<T, f16>::value;

// The largest over aligned groups of W lanes, every lane gets it (as group_sum)
template <int W>
__device__ __forceinline__ float group_max(float v) {
  auto moved = [](float x, auto ctrl) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  v = fmaxf(v, moved(v, std::integral_constant<int, 0xB1>{}));
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x4E>{}));
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x141>{}));
  v = fmaxf(v, moved(v, std::integral_constant<int, 0x140>{}));
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  return W == 64 ? with_other_half(v) : v;
}
__device__ __forceinline__ float uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

template <typename F>
__device__ __forceinline__ float square(const F& x, float s = 0.f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf((float)x[j], (float)x[j], s);
  return s;
}

// The power of two that brings values up to `bound` to at most 2^14 (what is not finite is left as it is)
__device__ __forceinline__ int to_range(float bound) { return bound > 0.f && bound < INFINITY ? 13 - ilogbf(bound) : 0; }

// For every key head, in parts of its keys and rows: the largest |v_j|^2 of keys that are seen, and |dout_i|^2 of rows that see any
template <typename T, int D>
__global__ __launch_bounds__(256) void diff_attn_sizes(DiffArgs a) {
  using F = typename Frag8<T>::type;
  constexpr int L = 2 * D / 8, kRows = 256 / L;                                // threads of a row, eight values each; rows at a time, four times
  __shared__ float2 most[4];
  const int tid = threadIdx.x, group = tid / L, e = tid % L * 8;
  for (long long at_part = blockIdx.x; at_part < (long long)a.B * a.Hk * a.size_parts; at_part += gridDim.x) {
    const int bh = (int)(at_part / a.size_parts), part = (int)(at_part % a.size_parts), b = bh / a.Hk, hk = bh % a.Hk;
    const int keys = (a.M + a.size_parts - 1) / a.size_parts, k0 = part * keys, k1 = min(k0 + keys, a.M);
    const int all = a.N * a.G, rows = (all + a.size_parts - 1) / a.size_parts, r0 = part * rows, r1 = min(r0 + rows, all);
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
    const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh + e;
    float v2 = 0.f, g2 = 0.f;
    for (int k = k0 + group; k < k1; k += 4 * kRows) {
      F x[4];
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = min(k + j * kRows, k1 - 1);
        x[j] = load8<T>(v + at * a.v_sn);
        in[j] = !mask || mask[at];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = group_sum<L>(square(x[j]));
        v2 = in[j] ? fmaxf(v2, s) : v2;
      }
    }
    for (int r = r0 + group; r < r1; r += 4 * kRows) {
      F x[4];
      float lse[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = min(r + j * kRows, r1 - 1), n = at / a.G, head = hk * a.G + at % a.G;
        x[j] = load8<T>((const T*)a.dout + (((long long)b * a.N + n) * a.H + head) * 2 * D + e);
        lse[j] = a.lse[((long long)b * a.H + head) * 2 * a.N + n];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = group_sum<L>(square(x[j]));
        g2 = lse[j] == INFINITY ? g2 : fmaxf(g2, s);
      }
    }
    v2 = group_max<64>(v2);
    g2 = group_max<64>(g2);
    if ((tid & 63) == 0) most[tid >> 6] = make_float2(v2, g2);
    __syncthreads();
    if (tid == 0)
      *(float2*)(a.sizes + 2 * at_part) = make_float2(fmaxf(fmaxf(most[0].x, most[1].x), fmaxf(most[2].x, most[3].x)),
                                                           fmaxf(fmaxf(most[0].y, most[1].y), fmaxf(most[2].y, most[3].y)));
    __syncthreads();
  }
}

// The largest |lam| of the heads that share a key head
template <typename T>
__device__ __forceinline__ float largest_lam(const DiffArgs& a, int hk, int lane) {
  float lam = 0.f;
  for (int u = lane; u < a.G; u += 64) lam = fmaxf(lam, fabsf(lam_of<T>(a, hk * a.G + u)));
  return group_max<64>(lam);
}

// A key head's largest |v_j|^2, and the powers of two of its score gradients (the second map's with lam) and of a1 - lam a2
struct Range { float v2; int grad, map; };
template <typename T>
__device__ __forceinline__ Range range_of(const DiffArgs& a, int bh, int hk, int lane) {
  float2 e = make_float2(0.f, 0.f);
  for (int i = lane; i < a.size_parts; i += 64) {
    const float2 x = *(const float2*)(a.sizes + ((long long)bh * a.size_parts + i) * 2);
    e = make_float2(fmaxf(e.x, x.x), fmaxf(e.y, x.y));
  }
  const float lam = largest_lam<T>(a, hk, lane), v2 = group_max<64>(e.x), g2 = group_max<64>(e.y);
  return {uniform(v2), __builtin_amdgcn_readfirstlane(to_range(2.f * sqrtf(v2 * g2) * fmaxf(lam, 1.f))), __builtin_amdgcn_readfirstlane(to_range(1.f + lam))};
}

template <typename T, int D, bool MORE = true> struct BwdShape {               // MORE: dq or dk is formed
  static constexpr bool kWeave = sizeof(T) == 2 && D == 128 && MORE;
  static constexpr int kMinWaves = sizeof(T) == 2 && !kWeave ? 2 : 1;
  static constexpr bool kLdsV = sizeof(T) == 2 && D == 64;                     // dk, dv: the wave's own values stay in LDS, to keep two waves on a SIMD
};

// Bit row_of(i, 0): whether value i of a lane, row row_of(i, h) of its block, is one of rows lo .. hi
__device__ __forceinline__ unsigned rows_of_lane(int lo, int hi, int h) {
  const unsigned upto = hi >= 31 ? ~0u : hi < 0 ? 0u : (2u << hi) - 1, below = lo > 31 ? ~0u : lo <= 0 ? 0u : (1u << lo) - 1;
  return (upto & ~below) >> (4 * h);
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, (BwdShape<T, D>::kMinWaves)) void diff_attn_dq(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  constexpr bool kWeave = BwdShape<T, D>::kWeave;
  constexpr int KT = 32, NK = D / 16, NV = 2 * D / 16, NC = D / 32, KR = kWeave ? 4 : 2;   // KR: blocks of k in LDS
  constexpr int kTile = KT * TL::kRow;
  __shared__ __attribute__((aligned(1024))) char tiles_lds[(KR + 2) * kTile];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const typename TL::Lane at(lane);
  const int rows = a.N * a.G, tiles = (rows + NW * 32 - 1) / (NW * 32);
  unsigned id = by_xcd(blockIdx.x, gridDim.x);
  const int share = id % a.q_shares;
  id /= a.q_shares;
  const int tile = tiles - 1 - (int)(id % tiles);
  const int bh = id / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int len = a.M;
  const int r0 = (tile * NW + wave) * 32, r = r0 + (lane & 31), rc = min(r, rows - 1);
  const int n = rc / a.G, head = hk * a.G + rc % a.G;
  const int off = len - a.N;
  const int lim = r >= rows ? -1 : a.causal ? min(n + off, len - 1) : len - 1;
  const int lim_lo = r0 + 31 >= rows ? -1 : a.causal ? min(r0 / a.G + off, len - 1) : len - 1;
  const int wg_hi = a.causal ? min(min((tile + 1) * NW * 32 - 1, rows - 1) / a.G + off, len - 1) : len - 1;
  const int all = max((wg_hi + KT) / KT, 0), per = (all + a.q_shares - 1) / a.q_shares, t0 = share * per, t1 = min(all, t0 + per);
  const long long oat = ((long long)b * a.N + n) * a.H + head;

  const T* q = (const T*)a.q + b * a.q_sb + n * a.q_sn + head * a.q_sh + 8 * h;
  const T* go = (const T*)a.dout + oat * 2 * D + 8 * h;
  F qf[2][NK], gf[NV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[m][s] = load8<T>(q + m * a.q_sm + 16 * s);
#pragma unroll
  for (int s = 0; s < NV; ++s) gf[s] = load8<T>(go + 16 * s);
  float delta[2] = {0.f, 0.f}, lse[2];
  const long long st = ((long long)b * a.H + head) * 2 * a.N + n;
#pragma unroll
  for (int m = 0; m < 2; ++m) lse[m] = a.lse[st + m * a.N];
  if (lse[0] == INFINITY)                                                      // a row that sees nothing is 0 whatever its gradient holds (in f16, often an overflow)
#pragma unroll
    for (int s = 0; s < NV; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) gf[s][j] = (T)0.f;
  if (a.o12) {
    const float* oo = a.o12 + oat * 4 * D + 8 * h;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < NV; ++s) {
        const Frag8<float>::type e = load8<float>(oo + m * 2 * D + 16 * s);
#pragma unroll
        for (int j = 0; j < 8; ++j) delta[m] = fmaf((float)gf[s][j], e[j], delta[m]);
      }
  }
  const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
  const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  f32x16 dq[2][NC], s[2], g;
  F ds[2][2];
  float dlam = 0.f;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int c = 0; c < NC; ++c) dq[m][c] = zero16();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ds[m][i][j] = (T)0.f;
  }
  const typename TL::template Loader<KT, NW> lk(a.k_sn, a.k_sm, tid), lv(a.v_sn, D, tid);
  auto ktile = [&](int t) { return tiles_lds + (t & (KR - 1)) * kTile; };
  auto vtile = [&](int t) { return tiles_lds + (KR + (t & 1)) * kTile; };
  auto fetch = [&](int t) {
    lk(ktile(t), k + (long long)t * KT * a.k_sn, len - t * KT, tid, wave);
    lv(vtile(t), v + (long long)t * KT * a.v_sn, len - t * KT, tid, wave);
  };
  auto seen_of = [&](int t) { return mask || t * KT + KT > len ? (unsigned)keys_seen<KT>(mask, t * KT, len, lane) : ~0u; };
  auto form = [&](f32x16 (&s_)[2], f32x16& g_, int t) {
    const char *kb = ktile(t), *vb = vtile(t);
    s_[0] = s_[1] = g_ = zero16();
    weave<F, 2 * NK + NV, 2>([&](int i) { return i < 2 * NK ? TL::row(kb, at, (i & 1) * NK + i / 2) : TL::row(vb, at, i - 2 * NK); },
                             [&](int i, const F& f) {
                               if (i < 2 * NK) s_[i & 1] = mma(f, qf[i & 1][i / 2], s_[i & 1]);
                               else g_ = mma(f, gf[i - 2 * NK], g_);
                             },
                             [](int) {});
  };
  auto hide = [&](unsigned seen, int t) {                                      // masked keys of block t: their probability becomes 0
    if (seen != ~0u || t * KT + 31 > lim_lo) {
      const unsigned ok = keys_of_lane(seen, lim - t * KT, h);
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m) s[m][i] = (ok >> row_of(i, 0)) & 1 ? s[m][i] : -INFINITY;
    }
  };
  auto turn = [&]() {                                                          // scores to score gradients (the second map's without its -lam)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][i], a.c, -lse[0])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][i], a.c, -lse[1]));
      dlam = fmaf(p1, g[i], dlam);
      s[0][i] = p0 * (g[i] - delta[0]);
      s[1][i] = p1 * (g[i] - delta[1]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) ds[m][i] = pack<T>(s[m], i);
  };
  auto add = [&](int t) {
    const char* kb = ktile(t);
    weave<F, 4 * NC, 2>([&](int i) { return TL::col(kb, at, i / (2 * NC), i % (2 * NC)); },
                        [&](int i, const F& f) {
                          const int c = i % (2 * NC);
                          dq[c / NC][c % NC] = mma(f, ds[c / NC][i / (2 * NC)], dq[c / NC][c % NC]);
                        },
                        [](int) {});
  };
  auto clean = [&](unsigned seen, int t) {                                     // what stands in masked keys may be anything, and 0 * NaN is NaN
    if (seen != ~0u) {
      TL::template clear<KT, NW * 64>(ktile(t), seen, tid);
      TL::template clear<KT, NW * 64>(vtile(t), seen, tid);
      __syncthreads();
    }
  };
  // Blocks first .. last - 1, one after the other
  auto sweep = [&](int first, int last, auto work) {
    if (first >= last) return;
    fetch(first);
    unsigned seen = seen_of(first);
    fetched();
    if (first + 1 < last) fetch(first + 1);
    clean(seen, first);
    for (int t = first; t < last; ++t) {
      form(s, g, t);
      hide(seen, t);
      work(t);
      if (t + 1 < last) {
        seen = seen_of(t + 1);
        fetched();
        if (t + 2 < last) fetch(t + 2);
        clean(seen, t + 1);
      }
    }
    __syncthreads();                                                           // (the tiles are read)
  };
  // delta = dout . o_i = sum of A_i G: without the maps' outputs, from one more sweep over the keys
  if (!a.o12)
    sweep(0, all, [&](int) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) delta[m] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[m][i], a.c, -lse[m])), g[i], delta[m]);
    });
  int ranged = 0;                                                              // the power of two of the row's score gradients
  float kept[2] = {1.f, 1.f};                                                  // delta is kept times what the key head's are brought into range by
  if constexpr (kRanged<T>) {
    const Range range = range_of<T>(a, bh, hk, lane);
    kept[0] = ldexpf(1.f, range.grad);
    kept[1] = ldexpf(1.f, range.grad - range.map);
    float g2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) g2 = square(gf[i], g2);
    g2 += __shfl_xor(g2, 32, 64);
    ranged = to_range(2.f * sqrtf(range.v2 * g2));
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    delta[m] += __shfl_xor(delta[m], 32, 64);
    if (h == 0 && r < rows && share == 0) a.delta[st + m * a.N] = delta[m] * kept[m];
    if constexpr (kRanged<T>) lse[m] -= (float)ranged;                         // (probabilities, and with them all that follows, times this power of two)
  }
  if constexpr (!kWeave) {
    sweep(t0, t1, [&](int t) {
      turn();
      add(t);
    });
  } else if (t0 < t1) {
    fetch(t0);
    unsigned seen = seen_of(t0);
    for (int i = tid; i < kTile / 16; i += NW * 64) *(float4*)(ktile(t0 - 1) + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);   // (its score gradients are 0)
    fetched();
    if (t0 + 1 < t1) fetch(t0 + 1);
    clean(seen, t0);
    form(s, g, t0);
    for (int t = t0; t < t1; ++t) {
      const unsigned next = t + 1 < t1 ? seen_of(t + 1) : ~0u;
      fetched();                                                       // block t + 1 has come; nobody reads k of t - 2 or v of t any more
      if (t + 2 < t1) fetch(t + 2);
      clean(next, t + 1);
      hide(seen, t);
      f32x16 s2[2] = {zero16(), zero16()}, g2 = zero16();
      const char *kn = ktile(t + 1), *vn = vtile(t + 1), *kb = ktile(t - 1);   // (behind the last block: whatever stands there, unused)
      F dn[2][2];
      constexpr int NS = 2 * NK, NG = NS + NV, NP = NG + 4 * NC;
      weave<F, NP, 3>(
          [&](int i) {
            return i < NS ? TL::row(kn, at, (i & 1) * NK + i / 2) : i < NG ? TL::row(vn, at, i - NS)
                                                                                      : TL::col(kb, at, (i - NG) / (2 * NC), (i - NG) % (2 * NC));
          },
          [&](int i, const F& f) {
            if (i < NS) s2[i & 1] = mma(f, qf[i & 1][i / 2], s2[i & 1]);
            else if (i < NG) g2 = mma(f, gf[i - NS], g2);
            else {
              const int c = (i - NG) % (2 * NC);
              dq[c / NC][c % NC] = mma(f, ds[c / NC][(i - NG) / (2 * NC)], dq[c / NC][c % NC]);
            }
          },
          [&](int i) {
#pragma unroll
            for (int x = 16 * i / NP; x < 16 * (i + 1) / NP; ++x) {
              const float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][x], a.c, -lse[0])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][x], a.c, -lse[1]));
              dlam = fmaf(p1, g[x], dlam);
              dn[0][x / 8][x % 8] = (T)(p0 * (g[x] - delta[0]));
              dn[1][x / 8][x % 8] = (T)(p1 * (g[x] - delta[1]));
            }
          });
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        ds[m][0] = dn[m][0];
        ds[m][1] = dn[m][1];
        s[m] = s2[m];
      }
      asm volatile("" : "+v"(g2));                                           // (or its products are moved behind the others, to where they are used)
      g = g2;
      seen = next;
    }
    add(t1 - 1);
  }
  landed();
  const float undo = ldexpf(1.f, -ranged);
  if constexpr (kRanged<T>) dlam *= undo;
  dlam += __shfl_xor(dlam, 32, 64);
  if (r >= rows) dlam = 0.f;
  if ((a.G & (a.G - 1)) == 0 && a.G <= 32) {                                   // one value for each head of the wave
    for (int o = 16; o >= a.G; o >>= 1) dlam += __shfl_xor(dlam, o, 64);
    if (lane < a.G) a.dlam_part[(((long long)bh * tiles + tile) * a.q_shares + share) * NW * a.G + wave * a.G + lane] = dlam;
  } else if (r < rows && h == 0) {
    a.dlam_part[((long long)bh * a.q_shares + share) * rows + r] = dlam;
  }
  if (r < rows && a.dq) {
    T* out = (T*)a.dq + oat * 2 * D + 4 * h;
    float* part = a.dq_part + ((long long)share * a.B * a.N * a.H + oat) * 2 * D + 4 * h;
    float f[2] = {a.scale, -lam_of<T>(a, head) * a.scale};
    if constexpr (kRanged<T>) {
      f[0] *= undo;
      f[1] *= undo;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float w[4] = {dq[m][c][4 * u] * f[m], dq[m][c][4 * u + 1] * f[m], dq[m][c][4 * u + 2] * f[m], dq[m][c][4 * u + 3] * f[m]};
          if (a.q_shares > 1) store4<float>(part + m * D + 32 * c + 8 * u, w[0], w[1], w[2], w[3]);
          else store4<T>(out + m * D + 32 * c + 8 * u, w[0], w[1], w[2], w[3]);
        }
  }
}

// DK, DV: which of the two this launch forms.  At D = 128 their sums and the keys' own values do not fit a wave's registers together, and the scores are formed twice.
template <typename T, int D, int NW, bool DK, bool DV>
__global__ __launch_bounds__(NW * 64, (BwdShape<T, D, DK>::kMinWaves)) void diff_attn_dkv(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  constexpr bool kWeave = BwdShape<T, D, DK>::kWeave;
  constexpr int QT = 32, NK = D / 16, NV = DK ? 2 * D / 16 : 1, NC = DK ? D / 32 : 1, ND = DV ? 2 * D / 32 : 1, R = kWeave ? 4 : 2;   // R: blocks in LDS
  constexpr int kTile = QT * TL::kRow;
  constexpr bool kLdsV = BwdShape<T, D>::kLdsV && DK;
  __shared__ __attribute__((aligned(1024))) char tiles_lds[(2 * R + (kLdsV ? NW : 0)) * kTile];
  __shared__ __attribute__((aligned(16))) float stat[R][4][QT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const typename TL::Lane at(lane);
  const int tiles = (a.M + NW * 32 - 1) / (NW * 32);
  unsigned id = by_xcd(blockIdx.x, gridDim.x);
  const int share = id % a.kv_shares;
  id /= a.kv_shares;
  const int tile = (int)(id % tiles), bh = id / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int off = a.M - a.N;
  const int k0 = (tile * NW + wave) * 32, key = k0 + (lane & 31), kc = min(key, a.M - 1);
  const T* k = (const T*)a.k + b * a.k_sb + kc * a.k_sn + hk * a.k_sh + 8 * h;
  const T* v = (const T*)a.v + b * a.v_sb + kc * a.v_sn + hk * a.v_sh + 8 * h;
  const bool seen = key < a.M && (!a.mask || a.mask[b * a.mask_sb + kc]);
  F kf[2][NK], vf[kLdsV ? 1 : NV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < NK; ++s) kf[m][s] = load8<T>(k + m * a.k_sm + 16 * s);
  const char* own_v = tiles_lds + (2 * R + wave) * kTile;
  if constexpr (kLdsV) {
    const typename TL::template Loader<NW * 32, NW> lv(a.v_sn, D, tid);
    lv(tiles_lds + 2 * R * kTile, (const T*)a.v + b * a.v_sb + (long long)tile * NW * 32 * a.v_sn + hk * a.v_sh, a.M - tile * NW * 32, tid, wave);
  } else if constexpr (DK) {
#pragma unroll
    for (int s = 0; s < NV; ++s) vf[s] = load8<T>(v + 16 * s);
  }
  f32x16 dk[2][NC], dv[ND], s[2], g;
  F ds[2][2], pc[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int c = 0; c < NC; ++c) dk[m][c] = zero16();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) { ds[m][i][j] = (T)0.f; pc[i][j] = (T)0.f; }
  }
#pragma unroll
  for (int c = 0; c < ND; ++c) dv[c] = zero16();

  // Queries that see nothing stand in front of all others (they have no key at or before their place, or none at all), and have no part in any gradient, whatever they and
  // their own gradient hold (in f16, often an overflow): blocks of them are left out, and in the block where they end the first other row takes their places
  int blind = a.causal ? max(0, -off) : 0;
  if (a.mask) {
    const unsigned char* mask = a.mask + b * a.mask_sb;
    int key0 = 0;
    unsigned long long any = 0;
    for (; key0 < a.M; key0 += 256) {
      unsigned long long at4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) at4[i] = keys_seen<64>(mask, key0 + 64 * i, a.M, lane);
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (at4[i]) { any = at4[i]; blind = key0 + 64 * i + __builtin_ctzll(at4[i]); }   // (the first key anyone sees)
      if (any) break;
    }
    blind = !any ? a.N : a.causal ? max(0, blind - off) : 0;
  }
  // f16: what brings the maps' difference (with lam), and each map's score gradients, into range (delta comes times x0 and x1)
  Range range = {0.f, 0, 0};
  if constexpr (kRanged<T>) range = range_of<T>(a, bh, hk, lane);
  const float pk = uniform(ldexpf(1.f, range.map)), x0 = uniform(ldexpf(1.f, range.grad)), x1 = uniform(ldexpf(1.f, range.grad - range.map));
  auto lam_ranged = [&](int head) { return kRanged<T> ? lam_of<T>(a, head) * pk : lam_of<T>(a, head); };
  auto apart = [&](float p0, float p1) { return kRanged<T> ? fmaf(p0, pk, -p1) : p0 - p1; };
  auto above = [&](float g_, float d, float x) { return kRanged<T> ? fmaf(g_, x, -d) : g_ - d; };
  // the blocks: queries that see the workgroup's first key, of each head that shares it
  const int first = max(blind, a.causal ? tile * NW * 32 - off : 0) / QT, nq = blind < a.N ? max((a.N + QT - 1) / QT - first, 0) : 0;
  const int all = nq * a.G, per = (all + a.kv_shares - 1) / a.kv_shares, from = min(share * per, all), total = min(all, from + per) - from;
  auto qtile = [&](int t) { return tiles_lds + (t & (R - 1)) * kTile; };
  auto gtile = [&](int t) { return tiles_lds + (R + (t & (R - 1))) * kTile; };
  const typename TL::template Loader<QT, NW> lq(a.q_sn, a.q_sm, tid), lg((long long)a.H * 2 * D, D, tid);
  // (divisions run in vector registers; what the fetches' bases come from has to be known to be the same in every lane)
  const int from_g = __builtin_amdgcn_readfirstlane(nq ? from / nq : 0), from_n = from - from_g * nq;
  int to_head = hk * a.G + from_g, to_n = (first + from_n) * QT;               // what the next fetch brings
  auto fetch = [&](int t) {
    const int head = to_head, n0 = to_n;
    to_n += QT;
    if (to_n >= a.N) { to_n = first * QT; ++to_head; }
    lq(qtile(t), (const T*)a.q + b * a.q_sb + head * a.q_sh + n0 * a.q_sn, a.N - n0, tid, wave, blind - n0);
    lg(gtile(t), (const T*)a.dout + (((long long)b * a.N + n0) * a.H + head) * 2 * D, a.N - n0, tid, wave, blind - n0);
    const long long st = ((long long)b * a.H + head) * 2 * a.N + n0;
    const unsigned off = ((unsigned)h * a.N + min(lane & 31, a.N - 1 - n0)) * 4u;
    for (int w = wave; w < 2; w += NW)                                         // lse of both maps, then delta of both: 32 values each
      fetch4((w == 0 ? a.lse : a.delta) + st, off, lds_address(&stat[t & (R - 1)][2 * w][0]));
  };
  auto form = [&](f32x16 (&s_)[2], f32x16& g_, int t) {
    const char *qb = qtile(t), *gb = gtile(t);
    s_[0] = s_[1] = zero16();
    weave<F, 2 * NK, 2>([&](int i) { return TL::row(qb, at, (i & 1) * NK + i / 2); }, [&](int i, const F& f) { s_[i & 1] = mma(f, kf[i & 1][i / 2], s_[i & 1]); },
                        [](int) {});
    if constexpr (DK) {
      g_ = zero16();
      F w[2];
      if constexpr (kLdsV) w[0] = TL::row(own_v, at, 0);
      weave<F, NV, 2>([&](int i) { return TL::row(gb, at, i); },
                      [&](int i, const F& f) {
                        if constexpr (kLdsV) {
                          if (i + 1 < NV) w[(i + 1) & 1] = TL::row(own_v, at, i + 1);
                          g_ = mma(f, w[i & 1], g_);
                        } else {
                          g_ = mma(f, vf[i], g_);
                        }
                      },
                      [](int) {});
    }
  };
  auto hide = [&](int n0) {                                                    // queries behind the last, and those that do not see the lane's key
    if (n0 + QT > a.N || (a.causal && k0 + 31 > n0 + off)) {
      const unsigned ok = rows_of_lane(a.causal ? key - off - n0 : 0, a.N - 1 - n0, h);
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m) s[m][i] = (ok >> row_of(i, 0)) & 1 ? s[m][i] : -INFINITY;
    }
  };
  auto turn = [&](int t, float lam) {                                          // (the second map's score gradients with lam, without the sign)
    const float(*e)[QT] = stat[t & (R - 1)];
    f32x16 p;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const int at_ = 8 * u + 4 * h;
      const f4 e0 = *(const f4*)&e[0][at_], e1 = *(const f4*)&e[1][at_], d0 = *(const f4*)&e[2][at_], d1 = *(const f4*)&e[3][at_];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = 4 * u + j;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][x], a.c, -e0[j])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][x], a.c, -e1[j])) * lam;
        p[x] = apart(p0, p1);
        if constexpr (DK) {
          s[0][x] = p0 * above(g[x], d0[j], x0);
          s[1][x] = p1 * above(g[x], d1[j], x1);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (DV) pc[i] = pack<T>(p, i);
      if constexpr (DK) {
        ds[0][i] = pack<T>(s[0], i);
        ds[1][i] = pack<T>(s[1], i);
      }
    }
  };
  auto add = [&](int t) {
    const char *qb = qtile(t), *gb = gtile(t);
    constexpr int NDV = DV ? 2 * ND : 0, NP = NDV + (DK ? 4 * NC : 0);
    weave<F, NP, 2>([&](int i) { return i < NDV ? TL::col(gb, at, i / ND, i % ND) : TL::col(qb, at, (i - NDV) / (2 * NC), (i - NDV) % (2 * NC)); },
                    [&](int i, const F& f) {
                      if (i < NDV) dv[i % ND] = mma(f, pc[i / ND], dv[i % ND]);
                      else {
                        const int c = (i - NDV) % (2 * NC);
                        dk[c / NC][c % NC] = mma(f, ds[c / NC][(i - NDV) / (2 * NC)], dk[c / NC][c % NC]);
                      }
                    },
                    [](int) {});
  };
  if (total > 0) {
    fetch(0);
    if constexpr (kWeave)
      for (int i = tid; i < kTile / 16; i += NW * 64) {                        // (block -1: its probabilities and score gradients are 0)
        *(float4*)(qtile(-1) + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);
        *(float4*)(gtile(-1) + i * 16) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    fetched();
    if (total > 1) fetch(1);
    int head = hk * a.G + from_g, n0 = (first + from_n) * QT;
    float lam = lam_ranged(head);
    auto step = [&]() {
      n0 += QT;
      if (n0 >= a.N && head + 1 < (hk + 1) * a.G) { n0 = first * QT; lam = lam_ranged(++head); }
    };
    if constexpr (kWeave) {
      form(s, g, 0);
      for (int t = 0; t < total; ++t) {
        fetched();                                                       // block t + 1 has come; nobody reads block t - 2 any more
        if (t + 2 < total) fetch(t + 2);
        hide(n0);
        const float lam_t = lam;
        step();
        f32x16 s2[2] = {zero16(), zero16()}, g2 = zero16();
        const char *qn = qtile(t + 1), *gn = gtile(t + 1), *qb = qtile(t - 1), *gb = gtile(t - 1);   // (behind the last block: whatever stands there, unused)
        const float(*e)[QT] = stat[t & (R - 1)];
        typedef float f4 __attribute__((ext_vector_type(4)));
        f4 st[4];
        F dn[2][2], pn[2];
        constexpr int NS = 2 * NK, NG = NS + (DK ? NV : 0), NDV = NG + (DV ? 2 * ND : 0), NP = NDV + (DK ? 4 * NC : 0);
        weave<F, NP, 3>(
            [&](int i) {
              return i < NS    ? TL::row(qn, at, (i & 1) * NK + i / 2)
                     : i < NG  ? TL::row(gn, at, i - NS)
                     : i < NDV ? TL::col(gb, at, (i - NG) / ND, (i - NG) % ND)
                               : TL::col(qb, at, (i - NDV) / (2 * NC), (i - NDV) % (2 * NC));
            },
            [&](int i, const F& f) {
              if (i < NS) s2[i & 1] = mma(f, kf[i & 1][i / 2], s2[i & 1]);
              else if (i < NG) g2 = mma(f, vf[i - NS], g2);
              else if (i < NDV) dv[(i - NG) % ND] = mma(f, pc[(i - NG) / ND], dv[(i - NG) % ND]);
              else {
                const int c = (i - NDV) % (2 * NC);
                dk[c / NC][c % NC] = mma(f, ds[c / NC][(i - NDV) / (2 * NC)], dk[c / NC][c % NC]);
              }
            },
            [&](int i) {
#pragma unroll
              for (int x = 16 * i / NP; x < 16 * (i + 1) / NP; ++x) {
                if (x % 4 == 0)
#pragma unroll
                  for (int y = 0; y < (DK ? 4 : 2); ++y) st[y] = *(const f4*)&e[y][2 * x + 4 * h];
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][x], a.c, -st[0][x % 4])), p1 = __builtin_amdgcn_exp2f(fmaf(s[1][x], a.c, -st[1][x % 4])) * lam_t;
                if constexpr (DV) pn[x / 8][x % 8] = (T)apart(p0, p1);
                if constexpr (DK) {
                  dn[0][x / 8][x % 8] = (T)(p0 * above(g[x], st[2][x % 4], x0));
                  dn[1][x / 8][x % 8] = (T)(p1 * above(g[x], st[3][x % 4], x1));
                }
              }
            });
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if constexpr (DV) pc[m] = pn[m];
          if constexpr (DK) {
            ds[m][0] = dn[m][0];
            ds[m][1] = dn[m][1];
          }
          s[m] = s2[m];
        }
        if constexpr (DK) {
          asm volatile("" : "+v"(g2));                                         // (or its products are moved behind the others, to where they are used)
          g = g2;
        }
      }
      add(total - 1);
    } else {
      for (int t = 0; t < total; ++t) {
        form(s, g, t);
        hide(n0);
        turn(t, lam);
        add(t);
        step();
        if (t + 1 < total) {
          fetched();
          if (t + 2 < total) fetch(t + 2);
        }
      }
    }
  }
  landed();                                                                    // (without a block to work on, the wave's own values may still be)
  if (key >= a.M) return;
  // (a key nobody sees has gradient 0; what its lanes hold came of values that may be anything, and stayed in their own columns)
  const long long oat = (((long long)b * a.M + key) * a.Hk + hk) * 2 * D + 4 * h;
  const long long poat = oat + (long long)share * a.B * a.M * a.Hk * 2 * D;
  auto put = [&](void* out, float* part, int at_, const f32x16& x, float f) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float w[4] = {seen ? x[4 * u] * f : 0.f, seen ? x[4 * u + 1] * f : 0.f, seen ? x[4 * u + 2] * f : 0.f, seen ? x[4 * u + 3] * f : 0.f};
      if (a.kv_shares > 1) store4<float>(part + poat + at_ + 8 * u, w[0], w[1], w[2], w[3]);
      else store4<T>((T*)out + oat + at_ + 8 * u, w[0], w[1], w[2], w[3]);
    }
  };
  if constexpr (DV)
#pragma unroll
    for (int c = 0; c < ND; ++c) put(a.dv, a.dv_part, 32 * c, dv[c], ldexpf(1.f, -range.map));
  if constexpr (DK)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c) put(a.dk, a.dk_part, m * D + 32 * c, dk[m][c], ldexpf(m ? -a.scale : a.scale, -range.grad));
}

// Sums over the 32 lanes of a half: lane l gets that of value l & 15 of a (l & 16: of b).  In every step a lane keeps one half of the values it has and gives the other
// to its partner, 77 operations where 32 sums of their own are 192.
__device__ __forceinline__ float sums_of_half(const f32x16& a, const f32x16& b, int lane) {
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[i]), __float_as_uint(b[i]), false, false);
    w[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  auto step = [&](int n, auto ctrl) {                                          // partners differ in the bit of lane that is n (and perhaps in lower ones)
    const bool upper = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? w[i + n] : w[i], give = upper ? w[i] : w[i + n];
      w[i] = keep + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(give), decltype(ctrl)::value, 0xf, 0xf, true));
    }
  };
  step(8, std::integral_constant<int, 0x128>{});                               // lane ^ 8
  step(4, std::integral_constant<int, 0x141>{});                               // lane ^ 7
  step(2, std::integral_constant<int, 0x4E>{});                                // lane ^ 2
  step(1, std::integral_constant<int, 0xB1>{});                                // lane ^ 1
  return w[0];
}

// All gradients of a key head with up to 64 keys in one go: a workgroup holds the keys, a wave 32 of them, and the queries of the head pass by once, so that scores, maps and
// the products with v are formed once (10 products of N M D where the two kernels above have 14, or 20 with delta's sweep) and every input is read once.  delta is the sum of
// a row's A G over the lanes and waves that hold its keys; score gradients go through LDS, turned round, to the sum over keys that is dq.  Bound by its chain of loads, products
// and stores with a wave on a SIMD (2048 rays x 4 heads x 64 samples, float, D = 32: 326 us, on an idle card 350, the matrix pipe busy for 40%; three workgroups to a CU, or starts apart from each
// other, were no quicker).
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 1) void diff_attn_short(DiffArgs a) {
  using TL = Tile<T, D>;
  using F = typename Frag8<T>::type;
  constexpr int QT = 32, NK = D / 16, NV = 2 * D / 16, NC = D / 32, ND = 2 * D / 32, R = 2;
  constexpr int kTile = QT * TL::kRow, kPitch = NW * 32 + 8;                   // (the pitch keeps the writes of neighbouring rows in other banks)
  typedef T t4 __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(1024))) char tiles_lds[(2 * R + NW) * kTile];
  __shared__ __attribute__((aligned(16))) T turned[2][QT][kPitch];             // score gradients: [map][query][key]
  __shared__ __attribute__((aligned(16))) float stat[R][2][QT], sums[NW][2][QT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const typename TL::Lane at(lane);
  const int bh = (int)by_xcd(blockIdx.x, gridDim.x), b = bh / a.Hk, hk = bh % a.Hk, off = a.M - a.N;
  const int k0 = wave * 32, key = k0 + (lane & 31), kc = min(key, a.M - 1);
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const unsigned long long seen64 = keys_seen<NW * 32>(mask, 0, a.M, lane);
  const bool seen = (seen64 >> key) & 1;
  const unsigned seen32 = (unsigned)(seen64 >> k0);
  char* ktile = tiles_lds + 2 * R * kTile;
  const T* kbase = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
  const typename TL::template Loader<NW * 32, NW> lk(a.k_sn, a.k_sm, tid);
  lk(ktile, kbase, a.M, tid, wave);
  F vf[NV];
  {
    const T* v = (const T*)a.v + b * a.v_sb + kc * a.v_sn + hk * a.v_sh + 8 * h;
#pragma unroll
    for (int s = 0; s < NV; ++s) vf[s] = load8<T>(v + 16 * s);
    if (!seen) {                                                               // what stands in masked keys may be anything, and 0 * NaN is NaN
#pragma unroll
      for (int s = 0; s < NV; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) vf[s][j] = (T)0.f;
    }
  }
  // queries that see nothing stand in front (see above)
  const int key0 = seen64 ? __builtin_ctzll(seen64) : 0, blind = !seen64 ? a.N : a.causal ? max(0, key0 - off) : 0;
  const int first = blind / QT, total = blind < a.N ? ((a.N + QT - 1) / QT - first) * a.G : 0;
  if (a.dq) {                                                                  // blocks of them are left out
    const int none = total ? first * QT : a.N, per = 2 * D / 4;
    for (int i = tid; i < none * a.G * per; i += NW * 64) {
      const int n = i / (a.G * per), e = i - n * a.G * per;
      store4<T>((T*)a.dq + (((long long)b * a.N + n) * a.H + hk * a.G) * 2 * D + 4 * e, 0.f, 0.f, 0.f, 0.f);
    }
  }
  f32x16 dk[2][NC], dv[ND], s[2], g;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) dk[m][c] = zero16();
#pragma unroll
  for (int c = 0; c < ND; ++c) dv[c] = zero16();
  float dlam = 0.f;

  auto qtile = [&](int t) { return tiles_lds + (t % R) * kTile; };
  auto gtile = [&](int t) { return tiles_lds + (R + t % R) * kTile; };
  const typename TL::template Loader<QT, NW> lq(a.q_sn, a.q_sm, tid), lg((long long)a.H * 2 * D, D, tid);
  int to_head = hk * a.G, to_n = first * QT;                                   // what the next fetch brings
  auto fetch = [&](int t) {
    const int head = to_head, n0 = to_n;
    to_n += QT;
    if (to_n >= a.N) { to_n = first * QT; ++to_head; }
    lq(qtile(t), (const T*)a.q + b * a.q_sb + head * a.q_sh + n0 * a.q_sn, a.N - n0, tid, wave, blind - n0);
    lg(gtile(t), (const T*)a.dout + (((long long)b * a.N + n0) * a.H + head) * 2 * D, a.N - n0, tid, wave, blind - n0);
    if (wave == 0)
      fetch4(a.lse + ((long long)b * a.H + head) * 2 * a.N + n0, ((unsigned)h * a.N + min(lane & 31, a.N - 1 - n0)) * 4u, lds_address(&stat[t % R][0][0]));
  };
  // f16: one power of two for all score gradients of the key head.  It is that of the first block's largest |dout_i|; where a block's is more
  // than twice as large, what was added up follows
  float v2 = 0.f, pk = 1.f, most_lam = 1.f;
  int map = 0, grad = 200;                                                     // (200: none yet)
  __shared__ float most[NW];
  if constexpr (kRanged<T>) {
    const float lam = largest_lam<T>(a, hk, lane);
    map = __builtin_amdgcn_readfirstlane(to_range(1.f + lam));
    pk = uniform(ldexpf(1.f, map));
    most_lam = fmaxf(lam, 1.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) v2 = square(vf[i], v2);
    v2 = group_max<32>(v2 + __shfl_xor(v2, 32, 64));
    if (lane == 0) most[wave] = v2;
  }
  if (total > 0) {
    fetch(0);
    int head = hk * a.G, n0 = first * QT;
    float lam = lam_of<T>(a, head);
    for (int t = 0; t < total; ++t) {
      fetched();                                                               // block t has come
      if (kRanged<T> && t == 0 && NW > 1) v2 = fmaxf(most[0], most[NW - 1]);
      if (t == 0 && seen64 != (NW == 2 ? ~0ull : 0xffffffffull)) {
        TL::template clear<NW * 32, NW * 64>(ktile, seen64, tid);
        __syncthreads();
      }
      if (t + 1 < total) fetch(t + 1);
      const char *qb = qtile(t), *gb = gtile(t);
      s[0] = s[1] = g = zero16();
      struct Two { F q, k; };
      weave<Two, 2 * NK, 1>([&](int i) { return Two{TL::row(qb, at, (i & 1) * NK + i / 2), TL::row(ktile + wave * kTile, at, (i & 1) * NK + i / 2)}; },
                            [&](int i, const Two& f) { s[i & 1] = mma(f.q, f.k, s[i & 1]); }, [](int) {});
      float g2 = 0.f;
      weave<F, NV, 2>([&](int i) { return TL::row(gb, at, i); },
                      [&](int i, const F& f) {
                        g = mma(f, vf[i], g);
                        if constexpr (kRanged<T>) g2 = square(f, g2);
                      },
                      [](int) {});
      float x0 = 1.f;
      if constexpr (kRanged<T>) {
        g2 = group_max<32>(g2 + __shfl_xor(g2, 32, 64));
        const int now = __builtin_amdgcn_readfirstlane(to_range(2.f * sqrtf(v2 * g2) * most_lam));
        if (now < grad - 1 && g2 > 0.f && g2 < INFINITY) {
          if (grad < 200) {
            const float down = ldexpf(1.f, now - grad);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int c = 0; c < NC; ++c) dk[m][c] *= down;
            dlam *= down;
          }
          grad = now;
        }
        x0 = uniform(ldexpf(1.f, grad < 200 ? grad : 0));
      }
      if (n0 + QT > a.N || seen32 != ~0u || (a.causal && k0 + 31 > n0 + off)) {
        const unsigned ok = seen ? rows_of_lane(a.causal ? key - off - n0 : 0, a.N - 1 - n0, h) : 0u;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int m = 0; m < 2; ++m) s[m][i] = (ok >> row_of(i, 0)) & 1 ? s[m][i] : -INFINITY;
      }
      F pc[2];
      {
        f32x16 p;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          typedef float f4 __attribute__((ext_vector_type(4)));
          const f4 e0 = *(const f4*)&stat[t % R][0][8 * u + 4 * h], e1 = *(const f4*)&stat[t % R][1][8 * u + 4 * h];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int x = 4 * u + j;
            s[0][x] = __builtin_amdgcn_exp2f(fmaf(s[0][x], a.c, -e0[j]));
            s[1][x] = __builtin_amdgcn_exp2f(fmaf(s[1][x], a.c, -e1[j]));
            p[x] = kRanged<T> ? fmaf(-lam * pk, s[1][x], s[0][x] * pk) : fmaf(-lam, s[1][x], s[0][x]);
          }
        }
        const float part = sums_of_half(s[0] * g, s[1] * g, lane);
        sums[wave][(lane >> 4) & 1][row_of(lane & 15, h)] = kRanged<T> ? part * x0 : part;
        pc[0] = pack<T>(p, 0);
        pc[1] = pack<T>(p, 1);
      }
      weave<F, 2 * ND, 2>([&](int i) { return TL::col(gb, at, i / ND, i % ND); }, [&](int i, const F& f) { dv[i % ND] = mma(f, pc[i / ND], dv[i % ND]); }, [](int) {});
      __syncthreads();
      F ds[2][2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        typedef float f4 __attribute__((ext_vector_type(4)));
        f4 d0 = *(const f4*)&sums[0][0][8 * u + 4 * h], d1 = *(const f4*)&sums[0][1][8 * u + 4 * h];
        if constexpr (NW > 1) {
          d0 += *(const f4*)&sums[1][0][8 * u + 4 * h];
          d1 += *(const f4*)&sums[1][1][8 * u + 4 * h];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int x = 4 * u + j;
          if (n0 + 8 * u + 4 * h + j < a.N) dlam += d1[j];
          if constexpr (kRanged<T>) {
            s[0][x] *= fmaf(g[x], x0, -d0[j]);
            s[1][x] *= lam * fmaf(g[x], x0, -d1[j]);
          } else {
            s[0][x] *= g[x] - d0[j];
            s[1][x] *= lam * (g[x] - d1[j]);                                   // (without the sign)
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ds[m][i] = pack<T>(s[m], i);
#pragma unroll
          for (int j = 0; j < 8; ++j) turned[m][row_of(8 * i + j, h)][key] = ds[m][i][j];
        }
      weave<F, 4 * NC, 2>([&](int i) { return TL::col(qb, at, i / (2 * NC), i % (2 * NC)); },
                          [&](int i, const F& f) {
                            const int c = i % (2 * NC);
                            dk[c / NC][c % NC] = mma(f, ds[c / NC][i / (2 * NC)], dk[c / NC][c % NC]);
                          },
                          [](int) {});
      __syncthreads();
      if (a.dq)
        for (int m = wave; m < 2; m += NW) {
          f32x16 dq[NC];
#pragma unroll
          for (int c = 0; c < NC; ++c) dq[c] = zero16();
#pragma unroll
          for (int i = 0; i < NW * 2; ++i) {
            const T* e = &turned[m][lane & 31][16 * i + 4 * h];
            const F w = __builtin_shufflevector(*(const t4*)e, *(const t4*)(e + 8), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int c = 0; c < NC; ++c) dq[c] = mma(TL::col(ktile, at, i, m * NC + c), w, dq[c]);
          }
          const int n = n0 + (lane & 31);
          const float f = kRanged<T> ? ldexpf(m ? -a.scale : a.scale, grad < 200 ? -grad : 0) : m ? -a.scale : a.scale;
          if (n < a.N) {
            T* out = (T*)a.dq + (((long long)b * a.N + n) * a.H + head) * 2 * D + m * D + 4 * h;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int u = 0; u < 4; ++u) store4<T>(out + 32 * c + 8 * u, dq[c][4 * u] * f, dq[c][4 * u + 1] * f, dq[c][4 * u + 2] * f, dq[c][4 * u + 3] * f);
          }
        }
      n0 += QT;
      if (n0 >= a.N) {                                                         // the head's last block
        dlam += __shfl_xor(dlam, 32, 64);
        if (tid == 0) a.dlam_part[(long long)bh * a.G + head - hk * a.G] = kRanged<T> ? ldexpf(dlam, grad < 200 ? -grad : 0) : dlam;
        dlam = 0.f;
        n0 = first * QT;
        if (t + 1 < total) lam = lam_of<T>(a, ++head);
      }
    }
  } else {
    for (int i = tid; i < a.G; i += NW * 64) a.dlam_part[(long long)bh * a.G + i] = 0.f;
  }
  landed();                                                                    // (without a block to work on, the keys may still be on their way)
  if (key >= a.M || !a.dk) return;
  const long long oat = (((long long)b * a.M + key) * a.Hk + hk) * 2 * D + 4 * h;
  auto put = [&](T* out, const f32x16& x, float f) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      store4<T>(out + 8 * u, seen ? x[4 * u] * f : 0.f, seen ? x[4 * u + 1] * f : 0.f, seen ? x[4 * u + 2] * f : 0.f, seen ? x[4 * u + 3] * f : 0.f);
  };
#pragma unroll
  for (int c = 0; c < ND; ++c) put((T*)a.dv + oat + 32 * c, dv[c], ldexpf(1.f, -map));
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) put((T*)a.dk + oat + m * D + 32 * c, dk[m][c], ldexpf(m ? -a.scale : a.scale, grad < 200 ? -grad : 0));
}

// Adds the shares of a gradient, in order; n a multiple of 4
template <typename T>
__global__ __launch_bounds__(256) void diff_attn_add(const float* part, T* out, long long n, int shares) {
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
    float4 v = *(const float4*)(part + i);
    for (int s = 1; s < shares; ++s) {
      const float4 w = *(const float4*)(part + s * n + i);
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    store4<T>(out + i, v.x, v.y, v.z, v.w);
  }
}

// dlam[h] = - the sum of what the waves (or rows) left for it, in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void diff_attn_dlam(DiffArgs a, int units) {
  __shared__ float s[16];
  const int head = blockIdx.x, hk = head / a.G, u = head % a.G;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const long long all = (long long)a.B * units;
  auto at = [&](long long i) { return a.dlam_part[((i / units * a.Hk + hk) * units + i % units) * a.G + u]; };
  long long i = threadIdx.x;
  for (; i + 3 * 1024 < all; i += 4 * 1024)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += at(i + j * 1024);
  for (; i < all; i += 1024) v[0] += at(i);
  const float w = group_sum<64>((v[0] + v[1]) + (v[2] + v[3]));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int j = 0; j < 16; ++j) t += s[j];
    if (a.lam_f32) ((float*)a.dlam)[head] = -t;
    else ((T*)a.dlam)[head] = (T)-t;
  }
}

}  // namespace tok
}  // namespace pgrf
