// Norms before and after a block, fused with the block's gate and residual scale, and their gradients.
//   u = Npost(y);  x' = x + s g (.) u;  z = Npre(x')
//   rms:   N(a) = a r w,               r = (mean(a^2) + eps)^-1/2
//   layer: N(a) = (a - m) r w + b,     m = mean(a), r = (mean((a - m)^2) + eps)^-1/2
// With h = the normalised value (a r or (a - m) r) and t = g w the gradient of a norm is r (t - [mean(t)] - h mean(t h)) (the bracket for
// layer only), of its weight the column sum of g h, of its bias the column sum of g.
//
// Both directions move each value once (4 or 6 values of traffic per element) and do ~14 / 24 operations on it, so memory bounds them: a row lives in
// the registers of TPR threads (NIT vectors of V values each), its sums are formed by lane exchanges (and 16 bytes of LDS where a row takes the whole
// workgroup), and the weights stay in registers over the rows a workgroup walks.  All arithmetic is float; x' is rounded once on its way out and z
// comes from the unrounded x'.  Column sums: one partial row per workgroup in float, added in the fixed order of the workgroups by a second launch,
// so gradients do not depend on scheduling.
#include "pgrf_experiments.h"
#include "token_common.h"

namespace pgrf {
namespace tok {

struct NormArgs {
  const void *x, *y, *gate, *pw, *pb, *qw, *qb;
  void *xo, *z;
  float* stats;                                    // [rows][4]: mean, r of y; mean, r of x'
  long long rows, rpg;                             // rpg: consecutive rows that share a row of the gate
  int C, layer, post, pre;
  float scale, eps;
  // backward
  const void *dxo, *dz;
  void *dx, *dy, *dgate;                           // dgate here: only where every row has its own gate row
  float* part;                                     // [chunks][5][C]: dpost_w, dpost_b, dpre_w, dpre_b, dgate
  long long span, rpc;                             // rows that may share a chunk (those of a gate row, or all); rows of a chunk
  int cpg;                                         // chunks of a span
  int want;                                        // bit k: quantity k of `part` is wanted
};

template <int TPR>
struct RowSum {                                     // sums over the TPR threads of a row
  float (*buf)[2][4];
  int turn = 0;
  __device__ explicit RowSum(float (*b)[2][4]) : buf(b) {}
  __device__ void two(float& a, float& b) {
    a = group_sum<(TPR < 64 ? TPR : 64)>(a);
    b = group_sum<(TPR < 64 ? TPR : 64)>(b);
    if constexpr (TPR > 64) {
      // two buffers in turn: whoever writes one a second time has passed the barrier behind every read of its first contents
      const int w = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) { buf[turn][0][w] = a; buf[turn][1][w] = b; }
      __syncthreads();
      a = (buf[turn][0][0] + buf[turn][0][1]) + (buf[turn][0][2] + buf[turn][0][3]);
      b = (buf[turn][1][0] + buf[turn][1][1]) + (buf[turn][1][2] + buf[turn][1][3]);
      turn ^= 1;
    }
  }
};

template <typename T, int V, int TPR, int NIT>
__device__ __forceinline__ void load_row(const void* p, long long at, int t, int C, Vec<T, V> (&v)[NIT]) {
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int c = (i * TPR + t) * V;
    if (c < C) {
      v[i] = load_vec<T, V>((const T*)p + at + c);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i].e[j] = (T)0.f;
    }
  }
}

template <typename T, int V, int TPR, int NIT>
__global__ __launch_bounds__(256) void block_norm_kernel(NormArgs a) {
  __shared__ float buf[2][2][4];
  RowSum<TPR> sum(buf);
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR, C = a.C;
  const float inv = 1.f / (float)C;
  Vec<T, V> pw[NIT], pb[NIT], qw[NIT], qb[NIT];
  if (a.pw) load_row<T, V, TPR, NIT>(a.pw, 0, t, C, pw);
  if (a.pb) load_row<T, V, TPR, NIT>(a.pb, 0, t, C, pb);
  if (a.qw) load_row<T, V, TPR, NIT>(a.qw, 0, t, C, qw);
  if (a.qb) load_row<T, V, TPR, NIT>(a.qb, 0, t, C, qb);
  for (long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (long long)gridDim.x * RPB) {
    const long long at = row * C;
    Vec<T, V> xv[NIT], yv[NIT], gv[NIT];
    load_row<T, V, TPR, NIT>(a.x, at, t, C, xv);
    if (a.y) load_row<T, V, TPR, NIT>(a.y, at, t, C, yv);
    if (a.gate) load_row<T, V, TPR, NIT>(a.gate, (a.rows >> 32 ? row / a.rpg : (unsigned)row / (unsigned)a.rpg) * C, t, C, gv);
    float h[NIT][V], st[4] = {0.f, 1.f, 0.f, 1.f};
    auto stats = [&](float& mean, float& r) {       // of h
      mean = 0.f;
      float s0 = 0.f, s1 = 0.f;
      if (a.layer) {
#pragma unroll
        for (int i = 0; i < NIT; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) s0 += h[i][j];
        sum.two(s0, s1);
        mean = s0 * inv;
      }
      s0 = s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = (i * TPR + t) * V < C ? h[i][j] - mean : 0.f;
          s0 = fmaf(d, d, s0);
        }
      sum.two(s0, s1);
      r = 1.f / sqrtf(fmaf(s0, inv, a.eps));
    };
    if (a.y) {
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (float)yv[i].e[j];
      if (a.post) stats(st[0], st[1]);
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float u = h[i][j];
          if (a.post) {
            u = (u - st[0]) * st[1];
            if (a.pw) u *= (float)pw[i].e[j];
            if (a.pb) u += (float)pb[i].e[j];
          }
          u *= a.scale;
          if (a.gate) u *= (float)gv[i].e[j];
          h[i][j] = (float)xv[i].e[j] + u;
        }
      if (a.xo) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          const int c = (i * TPR + t) * V;
          Vec<T, V> o;
#pragma unroll
          for (int j = 0; j < V; ++j) o.e[j] = (T)h[i][j];
          if (c < C) store_vec<T, V>((T*)a.xo + at + c, o);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (float)xv[i].e[j];
    }
    if (a.pre) {
      stats(st[2], st[3]);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = (i * TPR + t) * V;
        Vec<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float u = (h[i][j] - st[2]) * st[3];
          if (a.qw) u *= (float)qw[i].e[j];
          if (a.qb) u += (float)qb[i].e[j];
          o.e[j] = (T)u;
        }
        if (c < C) store_vec<T, V>((T*)a.z + at + c, o);
      }
    }
    if (a.stats && t == 0) *(float4*)(a.stats + row * 4) = make_float4(st[0], st[1], st[2], st[3]);
  }
}

// One workgroup = one chunk of rows inside one gate row, so the gate is a constant of the chunk (or every row has its own: rpg == 1).
template <typename T, int V, int TPR, int NIT, bool LAYER>
__global__ __launch_bounds__(256) void block_norm_bwd_kernel(NormArgs a) {
  constexpr int RPB = 256 / TPR;
  __shared__ float buf[2][2][4];
  __shared__ float col[RPB > 1 ? 256 * NIT * V : 1];
  RowSum<TPR> sum(buf);
  const int t = threadIdx.x % TPR, C = a.C;
  const float inv = 1.f / (float)C;
  const long long gr = blockIdx.x / a.cpg;
  const long long first = gr * a.span + (long long)(blockIdx.x % a.cpg) * a.rpc;
  long long last = first + a.rpc;
  if (last > (gr + 1) * a.span) last = (gr + 1) * a.span;
  if (last > a.rows) last = a.rows;
  const bool per_row = a.gate && a.rpg == 1;       // a gate row of its own per row: its gradient is written in place
  const bool own_gate = per_row && a.dgate;
  Vec<T, V> pw[NIT], pb[NIT], qw[NIT], gv[NIT];
  if (a.pw) load_row<T, V, TPR, NIT>(a.pw, 0, t, C, pw);
  if (a.pb) load_row<T, V, TPR, NIT>(a.pb, 0, t, C, pb);
  if (a.qw) load_row<T, V, TPR, NIT>(a.qw, 0, t, C, qw);
  if (a.gate && !per_row) load_row<T, V, TPR, NIT>(a.gate, gr * C, t, C, gv);
  float aw[NIT][V], ab[NIT][V], cw[NIT][V], cb[NIT][V];
#pragma unroll
  for (int i = 0; i < NIT; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) aw[i][j] = ab[i][j] = cw[i][j] = cb[i][j] = 0.f;
  // (the loop bounds are those of the workgroup: with TPR > 64 every thread meets every barrier)
  for (long long row0 = first; row0 < last; row0 += RPB) {
    const long long row = row0 + threadIdx.x / TPR;
    const bool live = row < last;
    if (RPB > 1 && !live) continue;
    const long long at = row * C;
    const float4 st = *(const float4*)(a.stats + row * 4);
    Vec<T, V> xv[NIT], yv[NIT], dxv[NIT], dzv[NIT];
    if (a.pre) load_row<T, V, TPR, NIT>(a.x, at, t, C, xv);
    if (a.y) load_row<T, V, TPR, NIT>(a.y, at, t, C, yv);
    if (a.dxo) load_row<T, V, TPR, NIT>(a.dxo, at, t, C, dxv);
    if (a.pre && a.dz) load_row<T, V, TPR, NIT>(a.dz, at, t, C, dzv);
    // (row, not row / rpg: rpg is 1 here)
    if (per_row) load_row<T, V, TPR, NIT>(a.gate, at, t, C, gv);
    float dh[NIT][V];
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) dh[i][j] = a.dxo ? (float)dxv[i].e[j] : 0.f;
    if (a.pre && a.dz) {
      // x' is formed again from x and y, unrounded: a rounded x' would put its rounding into the gradients of the norm behind it
      auto hat_of = [&](int i, int j) {
        float v = (float)xv[i].e[j];
        if (a.y) {
          float u = (float)yv[i].e[j];
          if (a.post) {
            u = (u - st.x) * st.y;
            if (a.pw) u *= (float)pw[i].e[j];
            if (a.pb) u += (float)pb[i].e[j];
          }
          u *= a.scale;
          if (a.gate) u *= (float)gv[i].e[j];
          v += u;
        }
        return (v - st.z) * st.w;
      };
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {               // (columns behind C: dz was loaded as 0)
          const float hat = hat_of(i, j), g = (float)dzv[i].e[j], tt = a.qw ? g * (float)qw[i].e[j] : g;
          if (LAYER) { s0 += tt; cb[i][j] += g; }
          s1 = fmaf(tt, hat, s1);
          cw[i][j] = fmaf(g, hat, cw[i][j]);
        }
      sum.two(s0, s1);
      s0 *= inv;
      s1 *= inv;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float hat = hat_of(i, j), g = (float)dzv[i].e[j], tt = a.qw ? g * (float)qw[i].e[j] : g;
          dh[i][j] += st.w * ((LAYER ? tt - s0 : tt) - hat * s1);
        }
    }
    if (a.dx) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = (i * TPR + t) * V;
        Vec<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.e[j] = (T)dh[i][j];
        if (c < C) store_vec<T, V>((T*)a.dx + at + c, o);
      }
    }
    if (a.y) {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        Vec<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool in = (i * TPR + t) * V < C;    // (behind C the gradient of the pre norm left something)
          const float d = in ? dh[i][j] : 0.f, gate = a.gate ? (float)gv[i].e[j] : 1.f;
          const float hat = a.post ? ((float)yv[i].e[j] - st.x) * st.y : (float)yv[i].e[j];
          const float w = a.pw ? (float)pw[i].e[j] : 1.f;
          const float ge = per_row ? gate * d : d;
          aw[i][j] = fmaf(ge, hat, aw[i][j]);
          if (LAYER) ab[i][j] += ge;
          if (own_gate) o.e[j] = (T)(a.scale * d * fmaf(hat, w, a.pb ? (float)pb[i].e[j] : 0.f));
          const float tt = a.scale * gate * d * w;
          if (LAYER) s0 += tt;
          s1 = fmaf(tt, hat, s1);
          dh[i][j] = tt;
        }
        const int c = (i * TPR + t) * V;
        if (own_gate && c < C) store_vec<T, V>((T*)a.dgate + at + c, o);
      }
      if (a.post) {
        sum.two(s0, s1);
        s0 *= inv;
        s1 *= inv;
      }
      if (a.dy) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          const int c = (i * TPR + t) * V;
          Vec<T, V> o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float hat = ((float)yv[i].e[j] - st.x) * st.y;
            o.e[j] = (T)(a.post ? st.y * ((LAYER ? dh[i][j] - s0 : dh[i][j]) - hat * s1) : dh[i][j]);
          }
          if (c < C) store_vec<T, V>((T*)a.dy + at + c, o);
        }
      }
    }
  }
  // the chunk's column sums: RPB rows side by side are added in LDS, in order
  auto across = [&](float (&v)[NIT][V]) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) col[(i * V + j) * 256 + threadIdx.x] = v[i][j];
      __syncthreads();
      if (threadIdx.x < TPR)
        for (int k = 1; k < RPB; ++k)
#pragma unroll
          for (int i = 0; i < NIT; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] += col[(i * V + j) * 256 + k * TPR + t];
    }
  };
  if (!a.want) return;
  const bool use_b = LAYER;
  if (a.y) across(aw);
  if (a.y && use_b) across(ab);
  if (a.pre) across(cw);
  if (a.pre && use_b) across(cb);
  if (threadIdx.x >= TPR) return;
  float* out = a.part + (long long)blockIdx.x * 5 * C;
#pragma unroll
  for (int i = 0; i < NIT; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (i * TPR + t) * V + j;
      if (c >= C) continue;
      const float gate = a.gate && !per_row ? (float)gv[i].e[j] : 1.f;
      if (a.want & 1) out[c] = a.scale * gate * aw[i][j];
      if (a.want & 2) out[C + c] = a.scale * gate * ab[i][j];
      if (a.want & 4) out[2 * C + c] = cw[i][j];
      if (a.want & 8) out[3 * C + c] = cb[i][j];
      if (a.want & 16) {
        const float w = a.pw ? (float)pw[i].e[j] : 1.f;
        // (without a norm the bias slot is empty and `ab` is 0)
        out[4 * C + c] = a.scale * (a.post ? fmaf(aw[i][j], w, a.pb ? (float)pb[i].e[j] * ab[i][j] : 0.f) : aw[i][j]);
      }
    }
}

// Adds the partial rows of a column: 64 columns x 4 shares of the chunks per workgroup; blockIdx.y = quantity (0..3) or 4 + gate row
template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* part, long long chunks, int cpg, int C, void* o0, void* o1, void* o2, void* o3,
                                                         void* o4) {
  __shared__ float s[4][64];
  const int k = blockIdx.y < 4 ? blockIdx.y : 4;
  void* o = k == 0 ? o0 : k == 1 ? o1 : k == 2 ? o2 : k == 3 ? o3 : o4;
  if (!o) return;
  const long long gr = (long long)blockIdx.y - 4, lo = k < 4 ? 0 : gr * cpg, n = k < 4 ? chunks : cpg;
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), share = threadIdx.x >> 6;
  float v = 0.f;
  if (c < C) {
    const float* p = part + ((lo * 5 + k) * C + c);
    float u[4] = {0.f, 0.f, 0.f, 0.f};
    long long i = share;
    for (; i + 12 < n; i += 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] += p[(i + 4 * j) * 5 * C];
    for (; i < n; i += 4) u[0] += p[i * 5 * C];
    v = (u[0] + u[1]) + (u[2] + u[3]);
  }
  s[share][threadIdx.x & 63] = v;
  __syncthreads();
  if (share == 0 && c < C) {
    const int x = threadIdx.x & 63;
    ((T*)o)[(k < 4 ? 0 : gr * C) + c] = (T)((s[0][x] + s[1][x]) + (s[2][x] + s[3][x]));
  }
}

// chunks: enough workgroups to fill the chip several times over, none across a gate row
static long long cut_rows(NormArgs& a, int rpb) {
  a.span = a.gate && a.rpg > 1 ? a.rpg : a.rows;
  const long long gates = a.rows / a.span;         // (check_norm: rows divide into gate rows)
  long long cpg = (1024 + gates - 1) / gates;
  const long long most = (a.span + rpb - 1) / rpb;
  if (cpg > most) cpg = most;
  a.rpc = (a.span + cpg - 1) / cpg;
  a.rpc = (a.rpc + rpb - 1) / rpb * rpb;
  a.cpg = (int)((a.span + a.rpc - 1) / a.rpc);
  return gates * a.cpg;
}

struct Shape { int v, tpr, nit; };

// A row takes as few threads as hold it in one to four vectors each (up to 32 single values where rows start at any address): a wave then walks
// several rows at once and the sums stay inside it.  C = 1 024 in 16 bits: a wave per row with two vectors per lane.
static Shape shape_for(int C, int dtype, bool vec) {
  const int v = vec ? (dtype == PGRF_DTYPE_F32 ? 4 : 8) : 1;
  const int n = (C + v - 1) / v;
  if (vec) {
    if (n <= 4) return {v, 4, 1};
    if (n <= 16) return {v, 16, 1};
    if (n <= 64) return {v, 64, 1};
    if (n <= 128) return {v, 64, 2};
    if (n <= 256) return {v, 256, 1};
    if (n <= 512) return {v, 256, 2};
    if (n <= 1024) return {v, 256, 4};
    return {v, 256, 8};
  }
  if (n <= 16) return {1, 16, 1};
  if (n <= 64) return {1, 16, 4};
  if (n <= 256) return {1, 64, 4};
  if (n <= 1024) return {1, 256, 4};
  return {1, 256, 32};
}

static bool rows_vectorise(int C, int dtype, const void* const* ps, int n) {
  if (C % (dtype == PGRF_DTYPE_F32 ? 4 : 8)) return false;
  for (int i = 0; i < n; ++i)
    if (ps[i] && !aligned16(ps[i])) return false;
  return true;
}

template <typename T, int V, int TPR, int NIT>
static void run_norm(const NormArgs& a, long long chunks, bool bwd, hipStream_t s) {
  if (bwd) {
    if (a.layer) hipLaunchKernelGGL((block_norm_bwd_kernel<T, V, TPR, NIT, true>), dim3((unsigned)chunks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<T, V, TPR, NIT, false>), dim3((unsigned)chunks), dim3(256), 0, s, a);
    return;
  }
  const long long need = (a.rows + 256 / TPR - 1) / (256 / TPR);
  hipLaunchKernelGGL((block_norm_kernel<T, V, TPR, NIT>), dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, s, a);
}

template <typename T>
static void pick_norm(const NormArgs& a, const Shape& h, long long chunks, bool bwd, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
#define PGRF_NORM(VV, TT, NN) \
  if (h.v == VV && h.tpr == TT && h.nit == NN) return run_norm<T, VV, TT, NN>(a, chunks, bwd, s)
  PGRF_NORM(V, 4, 1);
  PGRF_NORM(V, 16, 1);
  PGRF_NORM(V, 64, 1);
  PGRF_NORM(V, 64, 2);
  PGRF_NORM(V, 256, 1);
  PGRF_NORM(V, 256, 2);
  PGRF_NORM(V, 256, 4);
  if constexpr (V == 4) { PGRF_NORM(V, 256, 8); }
  PGRF_NORM(1, 16, 1);
  PGRF_NORM(1, 16, 4);
  PGRF_NORM(1, 64, 4);
  PGRF_NORM(1, 256, 4);
  PGRF_NORM(1, 256, 32);
#undef PGRF_NORM
}

static void dispatch_norm(const NormArgs& a, int dtype, const Shape& h, long long chunks, bool bwd, hipStream_t s) {
  if (dtype == PGRF_DTYPE_F32) pick_norm<float>(a, h, chunks, bwd, s);
  else if (dtype == PGRF_DTYPE_BF16) pick_norm<bf16>(a, h, chunks, bwd, s);
  else pick_norm<f16>(a, h, chunks, bwd, s);
}

static int check_norm(const char* who, int dtype, long long rows, int C, int flags, long long rpg, const void* y, const void* gate) {
  if (!dtype_ok(dtype)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: dtype %d (PGRF_DTYPE_F32 | BF16 | F16)", who, dtype);
  if (C < 1 || C > PGRF_BLOCK_NORM_MAX_C) return set_error(PGRF_ERR_UNSUPPORTED, "%s: C=%d not in [1,%d]", who, C, PGRF_BLOCK_NORM_MAX_C);
  if (rows < 0 || rows > (1ll << 40)) return set_error(PGRF_ERR_ARG, "%s: rows=%lld", who, rows);
  if (flags & ~7) return set_error(PGRF_ERR_ARG, "%s: unknown flags %d", who, flags);
  if (!y && (gate || (flags & PGRF_NORM_POST))) return set_error(PGRF_ERR_ARG, "%s: a gate or a norm of y without y", who);
  if (!y && !(flags & PGRF_NORM_PRE)) return set_error(PGRF_ERR_ARG, "%s: neither y nor a norm of x: nothing to do", who);
  if (gate && (rpg < 1 || (rows && rows % rpg))) return set_error(PGRF_ERR_ARG, "%s: %lld rows do not divide into groups of %lld per gate row", who, rows, rpg);
  return PGRF_OK;
}

}  // namespace tok
}  // namespace pgrf

using namespace pgrf;
using namespace pgrf::tok;

extern "C" {

int pgrf_block_norm(const void* x, const void* y, const void* gate, long long rows_per_gate, const void* post_w, const void* post_b,
                    const void* pre_w, const void* pre_b, int dtype, long long rows, int C, int flags, float scale, float eps, void* x_out,
                    void* z_out, float* stats, void* stream) {
  const char* who = "pgrf_block_norm";
  int rc = check_norm(who, dtype, rows, C, flags, rows_per_gate, y, gate);
  if (rc) return rc;
  if (rows == 0) return PGRF_OK;
  if (!x || (y && !x_out) || ((flags & PGRF_NORM_PRE) && !z_out)) return set_error(PGRF_ERR_ARG, "%s: null x / x_out / z_out", who);
  if (stats && !aligned16(stats)) return set_error(PGRF_ERR_ARG, "%s: stats must be 16-byte aligned", who);
  NormArgs a = {};
  a.x = x; a.y = y; a.gate = gate; a.rpg = gate ? rows_per_gate : rows;
  a.post = (flags & PGRF_NORM_POST) ? 1 : 0; a.pre = (flags & PGRF_NORM_PRE) ? 1 : 0; a.layer = (flags & PGRF_NORM_LAYER) ? 1 : 0;
  a.pw = a.post ? post_w : nullptr; a.pb = a.post && a.layer ? post_b : nullptr;
  a.qw = a.pre ? pre_w : nullptr; a.qb = a.pre && a.layer ? pre_b : nullptr;
  a.xo = y ? x_out : nullptr; a.z = z_out; a.stats = stats; a.rows = rows; a.C = C; a.scale = scale; a.eps = eps;
  const void* ps[] = {x, y, gate, a.pw, a.pb, a.qw, a.qb, a.xo, a.pre ? z_out : nullptr};
  dispatch_norm(a, dtype, shape_for(C, dtype, rows_vectorise(C, dtype, ps, 9)), 0, false, (hipStream_t)stream);
  PGRF_TOK_LAUNCHED(who);
  return PGRF_OK;
}

size_t pgrf_block_norm_backward_workspace_bytes(long long rows, int C, long long rows_per_gate) {
  if (rows < 1 || C < 1 || rows_per_gate < 1) return 16;
  // an upper bound of cut_rows' chunks for every row split: at most 1 024 chunks plus one per gate row
  const long long gates = rows_per_gate > 1 ? (rows + rows_per_gate - 1) / rows_per_gate : 1;
  return (size_t)(1024 + gates) * 5 * (size_t)C * sizeof(float);
}

int pgrf_block_norm_backward(const void* x, const void* y, const void* gate, long long rows_per_gate, const void* post_w, const void* post_b,
                             const void* pre_w, const float* stats, const void* dx_out, const void* dz, int dtype, long long rows, int C, int flags,
                             float scale, void* dx, void* dy, void* dgate, void* dpost_w, void* dpost_b, void* dpre_w, void* dpre_b, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* who = "pgrf_block_norm_backward";
  int rc = check_norm(who, dtype, rows, C, flags, rows_per_gate, y, gate);
  if (rc) return rc;
  if (dgate && !gate) return set_error(PGRF_ERR_ARG, "%s: dgate without gate", who);
  NormArgs a = {};
  a.post = (flags & PGRF_NORM_POST) ? 1 : 0; a.pre = (flags & PGRF_NORM_PRE) ? 1 : 0; a.layer = (flags & PGRF_NORM_LAYER) ? 1 : 0;
  if (rows && (!stats || (a.pre && !x))) return set_error(PGRF_ERR_ARG, "%s: null stats / x", who);
  if (rows && !aligned16(stats)) return set_error(PGRF_ERR_ARG, "%s: stats must be 16-byte aligned", who);
  a.x = x; a.y = y; a.gate = gate; a.rpg = gate ? rows_per_gate : (rows ? rows : 1);
  a.pw = a.post ? post_w : nullptr; a.pb = a.post && a.layer ? post_b : nullptr; a.qw = a.pre ? pre_w : nullptr;
  a.stats = const_cast<float*>(stats); a.rows = rows; a.C = C; a.scale = scale;
  a.dxo = dx_out; a.dz = a.pre ? dz : nullptr; a.dx = dx; a.dy = y ? dy : nullptr;
  const bool per_row = gate && rows_per_gate == 1;
  a.dgate = per_row ? dgate : nullptr;
  a.part = (float*)workspace;
  a.want = (a.post && dpost_w ? 1 : 0) | (a.post && a.layer && dpost_b ? 2 : 0) | (a.pre && dpre_w ? 4 : 0) | (a.pre && a.layer && dpre_b ? 8 : 0) |
           (dgate && !per_row ? 16 : 0);
  const void* ps[] = {x, y, gate, a.pw, a.pb, a.qw, dx_out, dz, dx, dy, a.dgate};
  const Shape h = shape_for(C, dtype, rows_vectorise(C, dtype, ps, 11));
  long long chunks = 0;
  a.cpg = 1;
  const long long gates = (a.want & 16) && rows ? rows / rows_per_gate : 0;
  if (gates > 60000) return set_error(PGRF_ERR_UNSUPPORTED, "%s: %lld gate rows (at most 60000, or one for each row)", who, gates);
  if (rows) {
    chunks = cut_rows(a, 256 / h.tpr);
    if (a.want && (!workspace || workspace_bytes < (size_t)chunks * 5 * C * sizeof(float)))
      return set_error(PGRF_ERR_ARG, "%s: workspace too small (%zu < %zu bytes)", who, workspace_bytes, (size_t)chunks * 5 * C * sizeof(float));
    dispatch_norm(a, dtype, h, chunks, true, (hipStream_t)stream);
    PGRF_TOK_LAUNCHED(who);
  }
  if (a.want) {
    const dim3 grid((C + 63) / 64, 4 + (unsigned)gates);
    void *o0 = a.want & 1 ? dpost_w : nullptr, *o1 = a.want & 2 ? dpost_b : nullptr, *o2 = a.want & 4 ? dpre_w : nullptr,
         *o3 = a.want & 8 ? dpre_b : nullptr, *o4 = a.want & 16 ? dgate : nullptr;
#define PGRF_COLS(T) hipLaunchKernelGGL(column_sum_kernel<T>, grid, dim3(256), 0, (hipStream_t)stream, a.part, chunks, a.cpg, C, o0, o1, o2, o3, o4)
    if (dtype == PGRF_DTYPE_F32) PGRF_COLS(float);
    else if (dtype == PGRF_DTYPE_BF16) PGRF_COLS(bf16);
    else PGRF_COLS(f16);
#undef PGRF_COLS
    PGRF_TOK_LAUNCHED(who);
  }
  return PGRF_OK;
}

}  // extern "C"
