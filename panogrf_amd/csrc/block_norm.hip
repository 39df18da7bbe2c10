// Norms before and after a block, fused with the block's gate and residual scale, and their gradients.
//   u = Npost(y);  x' = x + s g (.) u;  z = Npre(x')
//   rms:   N(a) = a r w,               r = (mean(a^2) + eps)^-1/2
//   layer: N(a) = (a - m) r w + b,     m = mean(a), r = (mean((a - m)^2) + eps)^-1/2
// With h = the normalised value (a r or (a - m) r) and t = g w the gradient of a norm is r (t - [mean(t)] - h mean(t h)) (the bracket for
// layer only), of its weight the column sum of g h, of its bias the column sum of g.
//
// Both directions move each value once (4 or 6 values of traffic per element) and do ~14 / 24 operations on it, so memory bounds them: a row lives in
// the registers of TPR threads (NIT vectors of V values each), its sums are formed by lane exchanges (and through LDS where a row takes several
// waves), and the weights stay in registers over the rows a workgroup walks, each loaded while the one before is worked on.  All arithmetic is float; x' is rounded once on its way out and z
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
  int each;                                        // the gate is loaded for every row, not kept for a chunk
  int want;                                        // bit k: quantity k of `part` is wanted
};

// A row is held by TPR threads with eight values each (one vector of 16 bits' values, two of float's, eight single ones where rows start at any address), so that a
// wave's registers leave room for three others beside it; rows of up to 64 threads share a wave, longer ones take several and add up through LDS.
template <int TPR>
struct RowSum {
  float (*buf)[2][16];
  int turn = 0;
  __device__ explicit RowSum(float (*b)[2][16]) : buf(b) {}
  __device__ __forceinline__ void two(float& a, float& b) {
    a = group_sum<(TPR < 64 ? TPR : 64)>(a);
    b = group_sum<(TPR < 64 ? TPR : 64)>(b);
    if constexpr (TPR > 64) {
      // two buffers in turn: whoever writes one a second time has passed the barrier behind every read of its first contents
      constexpr int W = TPR / 64;
      const int w = threadIdx.x >> 6, w0 = w / W * W;
      if ((threadIdx.x & 63) == 0) { buf[turn][0][w] = a; buf[turn][1][w] = b; }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) { a += buf[turn][0][w0 + i]; b += buf[turn][1][w0 + i]; }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ float one(float a) {
    a = group_sum<(TPR < 64 ? TPR : 64)>(a);
    if constexpr (TPR > 64) {
      constexpr int W = TPR / 64;
      const int w = threadIdx.x >> 6, w0 = w / W * W;
      if ((threadIdx.x & 63) == 0) buf[turn][0][w] = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) a += buf[turn][0][w0 + i];
      turn ^= 1;
    }
    return a;
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

__device__ __forceinline__ long long gate_row(const NormArgs& a, long long row) {
  return a.rows >> 32 ? row / a.rpg : (long long)((unsigned)row / (unsigned)a.rpg);
}

template <typename T, int V, int TPR, int NIT>
__global__ __launch_bounds__((TPR > 256 ? TPR : 256), 4) void block_norm_kernel(NormArgs a) {
  constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
  __shared__ float buf[2][2][16];
  RowSum<TPR> sum(buf);
  const int t = threadIdx.x % TPR, C = a.C;
  const float inv = 1.f / (float)C;
  Vec<T, V> pw[NIT], pb[NIT], qw[NIT], qb[NIT];
  if (a.pw) load_row<T, V, TPR, NIT>(a.pw, 0, t, C, pw);
  if (a.pb) load_row<T, V, TPR, NIT>(a.pb, 0, t, C, pb);
  if (a.qw) load_row<T, V, TPR, NIT>(a.qw, 0, t, C, qw);
  if (a.qb) load_row<T, V, TPR, NIT>(a.qb, 0, t, C, qb);
  struct In { Vec<T, V> x[NIT], y[NIT], g[NIT]; };
  auto load = [&](In& r, long long row) {
    row = row < a.rows ? row : a.rows - 1;           // (a row behind the last: read again, not written)
    load_row<T, V, TPR, NIT>(a.x, row * C, t, C, r.x);
    if (a.y) load_row<T, V, TPR, NIT>(a.y, row * C, t, C, r.y);
    if (a.gate) load_row<T, V, TPR, NIT>(a.gate, gate_row(a, row) * C, t, C, r.g);
  };
  const long long step = (long long)gridDim.x * RPB;
  long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  In in;
  load(in, row);
  // (the workgroup's rows go together: with TPR > 64 every thread meets every barrier)
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.rows; row0 += step, row += step) {
    const long long at = row * C;
    const bool live = row < a.rows;
    In next;
    if (row0 + step < a.rows) load(next, row + step);   // (the next row is on its way while this one is worked on)
    float h[NIT][V], st[4] = {0.f, 1.f, 0.f, 1.f};
    auto stats = [&](float& mean, float& r) {       // of h
      mean = 0.f;
      if (a.layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NIT; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) s += (i * TPR + t) * V < C ? h[i][j] : 0.f;   // (behind C the norm of y left something)
        mean = sum.one(s) * inv;
      }
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = (i * TPR + t) * V < C ? h[i][j] - mean : 0.f;
          s = fmaf(d, d, s);
        }
      r = 1.f / sqrtf(fmaf(sum.one(s), inv, a.eps));
    };
    if (a.y) {
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (float)in.y[i].e[j];
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
          if (a.gate) u *= (float)in.g[i].e[j];
          h[i][j] = (float)in.x[i].e[j] + u;
        }
      if (live) {
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
        for (int j = 0; j < V; ++j) h[i][j] = (float)in.x[i].e[j];
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
        if (live && c < C) store_vec<T, V>((T*)a.z + at + c, o);
      }
    }
    if (a.stats && t == 0 && live) *(float4*)(a.stats + row * 4) = make_float4(st[0], st[1], st[2], st[3]);
    in = next;
  }
}

// One workgroup = one chunk of rows inside one gate row, so the gate is a constant of the chunk, or (`each`: every row has its own, or so many are shared that a chunk
// for each would be mostly partial sums, and no gradient of theirs is asked for) the gate is one more input of the row.
template <typename T, int V, int TPR, int NIT, bool LAYER>
__global__ __launch_bounds__((TPR > 256 ? TPR : 256), (TPR > 512 ? 4 : LAYER ? 2 : 3)) void block_norm_bwd_kernel(NormArgs a) {
  constexpr int WG = TPR > 256 ? TPR : 256, RPB = WG / TPR;
  __shared__ float buf[2][2][16];
  __shared__ float col[RPB > 1 ? WG * NIT * V : 1];
  RowSum<TPR> sum(buf);
  const int t = threadIdx.x % TPR, C = a.C;
  const float inv = 1.f / (float)C;
  const long long gr = blockIdx.x / a.cpg;
  const long long first = gr * a.span + (long long)(blockIdx.x % a.cpg) * a.rpc;
  long long last = first + a.rpc;
  if (last > (gr + 1) * a.span) last = (gr + 1) * a.span;
  if (last > a.rows) last = a.rows;
  const bool per_row = a.gate && a.each;
  const bool own_gate = per_row && a.dgate;        // a gate row of its own per row: its gradient is written in place
  Vec<T, V> pw[NIT], pb[NIT], qw[NIT], gv[NIT];
  if (a.pw) load_row<T, V, TPR, NIT>(a.pw, 0, t, C, pw);
  if (a.pb) load_row<T, V, TPR, NIT>(a.pb, 0, t, C, pb);
  if (a.qw) load_row<T, V, TPR, NIT>(a.qw, 0, t, C, qw);
  if (a.gate && !per_row) load_row<T, V, TPR, NIT>(a.gate, gr * C, t, C, gv);
  // column sums: in registers; where 1024 threads leave each too few of those, in LDS, every thread at its own places, and no second row is on its way either (bf16, 8192 rows
  // of 8192, layer: 241 us, 3.3 TB/s; with all of it in registers, spilled, 765)
  constexpr bool kLds = TPR > 512;
  __shared__ __attribute__((aligned(16))) float room[kLds ? (LAYER ? 4 : 2) * NIT * V * WG : 1];
  float aw[kLds ? 1 : NIT][V], ab[kLds ? 1 : NIT][V], cw[kLds ? 1 : NIT][V], cb[kLds ? 1 : NIT][V];
  enum { kAw, kCw, kAb, kCb };
  auto take = [&](float (&v)[V], float (&held)[kLds ? 1 : NIT][V], int k, int i) {
    if constexpr (kLds) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = room[((k * NIT + i) * TPR + t) * V + j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = held[i][j];
    }
  };
  auto give = [&](const float (&v)[V], float (&held)[kLds ? 1 : NIT][V], int k, int i) {
    if constexpr (kLds) {
#pragma unroll
      for (int j = 0; j < V; ++j) room[((k * NIT + i) * TPR + t) * V + j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) held[i][j] = v[j];
    }
  };
  {
    float zero[V];
#pragma unroll
    for (int j = 0; j < V; ++j) zero[j] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      give(zero, aw, kAw, i);
      give(zero, cw, kCw, i);
      if (LAYER) {
        give(zero, ab, kAb, i);
        give(zero, cb, kCb, i);
      }
    }
  }
  struct In { Vec<T, V> x[NIT], y[NIT], dx[NIT], dz[NIT], g[NIT]; float4 st; };
  auto load = [&](In& r, long long row) {
    row = row < last ? row : last - 1;               // (a row behind the chunk: read again, not counted)
    const long long at = row * C;
    r.st = *(const float4*)(a.stats + row * 4);
    if (a.pre && a.dz) {
      load_row<T, V, TPR, NIT>(a.x, at, t, C, r.x);
      load_row<T, V, TPR, NIT>(a.dz, at, t, C, r.dz);
    }
    if (a.y) load_row<T, V, TPR, NIT>(a.y, at, t, C, r.y);
    if (a.dxo) load_row<T, V, TPR, NIT>(a.dxo, at, t, C, r.dx);
    if (per_row) load_row<T, V, TPR, NIT>(a.gate, a.rpg == 1 ? at : gate_row(a, row) * C, t, C, r.g);
  };
  In in;
  long long row = first + threadIdx.x / TPR;
  if (first < last) load(in, row);
  // (the loop bounds are those of the workgroup: with TPR > 64 every thread meets every barrier)
  for (long long row0 = first; row0 < last; row0 += RPB, row += RPB) {
    const bool live = row < last;
    const long long at = row * C;
    In next;
    if (!kLds && row0 + RPB < last) load(next, row + RPB);   // (the next row is on its way while this one is worked on)
    const float4 st = in.st;
    auto gate_of = [&](int i, int j) { return a.gate ? (float)(per_row ? in.g[i].e[j] : gv[i].e[j]) : 1.f; };
    float dh[NIT][V];
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) dh[i][j] = a.dxo ? (float)in.dx[i].e[j] : 0.f;
    if (a.pre && a.dz) {
      // x' is formed again from x and y, unrounded: a rounded x' would put its rounding into the gradients of the norm behind it
      float hat[NIT][V], s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        float w[V], b[V];
        take(w, cw, kCw, i);
        if (LAYER) take(b, cb, kCb, i);
#pragma unroll
        for (int j = 0; j < V; ++j) {               // (columns behind C: dz was loaded as 0)
          float v = (float)in.x[i].e[j];
          if (a.y) {
            float u = (float)in.y[i].e[j];
            if (a.post) {
              u = (u - st.x) * st.y;
              if (a.pw) u *= (float)pw[i].e[j];
              if (a.pb) u += (float)pb[i].e[j];
            }
            u *= a.scale;
            if (a.gate) u *= gate_of(i, j);
            v += u;
          }
          hat[i][j] = (v - st.z) * st.w;
          const float g = live ? (float)in.dz[i].e[j] : 0.f, tt = a.qw ? g * (float)qw[i].e[j] : g;
          if (LAYER) { s0 += tt; b[j] += g; }
          s1 = fmaf(tt, hat[i][j], s1);
          w[j] = live ? fmaf(g, hat[i][j], w[j]) : w[j];   // (a row that counts twice may be NaN, and 0 * NaN is NaN)
        }
        give(w, cw, kCw, i);
        if (LAYER) give(b, cb, kCb, i);
      }
      if (LAYER) sum.two(s0, s1);
      else s1 = sum.one(s1);
      s0 *= inv;
      s1 *= inv;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float g = (float)in.dz[i].e[j], tt = a.qw ? g * (float)qw[i].e[j] : g;
          dh[i][j] += st.w * ((LAYER ? tt - s0 : tt) - hat[i][j] * s1);
        }
    }
    if (a.dx && live) {
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
        float sw[V], sb[V];
        take(sw, aw, kAw, i);
        if (LAYER) take(sb, ab, kAb, i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool in_row = (i * TPR + t) * V < C && live;    // (behind C the gradient of the pre norm left something)
          const float d = in_row ? dh[i][j] : 0.f, gate = gate_of(i, j);
          const float hat = a.post ? ((float)in.y[i].e[j] - st.x) * st.y : (float)in.y[i].e[j];
          const float w = a.pw ? (float)pw[i].e[j] : 1.f;
          const float ge = per_row ? gate * d : d;
          sw[j] = live ? fmaf(ge, hat, sw[j]) : sw[j];
          if (LAYER) sb[j] += ge;
          if (own_gate) o.e[j] = (T)(a.scale * d * fmaf(hat, w, a.pb ? (float)pb[i].e[j] : 0.f));
          const float tt = a.scale * gate * d * w;
          if (LAYER) s0 += tt;
          s1 = fmaf(tt, hat, s1);
          dh[i][j] = tt;
        }
        give(sw, aw, kAw, i);
        if (LAYER) give(sb, ab, kAb, i);
        const int c = (i * TPR + t) * V;
        if (own_gate && live && c < C) store_vec<T, V>((T*)a.dgate + at + c, o);
      }
      if (a.post) {
        if (LAYER) sum.two(s0, s1);
        else s1 = sum.one(s1);
        s0 *= inv;
        s1 *= inv;
      }
      if (a.dy && live) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          const int c = (i * TPR + t) * V;
          Vec<T, V> o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float hat = ((float)in.y[i].e[j] - st.x) * st.y;
            o.e[j] = (T)(a.post ? st.y * ((LAYER ? dh[i][j] - s0 : dh[i][j]) - hat * s1) : dh[i][j]);
          }
          if (c < C) store_vec<T, V>((T*)a.dy + at + c, o);
        }
      }
    }
    if constexpr (!kLds) in = next;
    else if (row0 + RPB < last) load(in, row + RPB);
  }
  // the chunk's column sums: RPB rows side by side are added in LDS, in order
  auto across = [&](auto& v) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) col[(i * V + j) * WG + threadIdx.x] = v[i][j];
      __syncthreads();
      if (threadIdx.x < TPR)
        for (int k = 1; k < RPB; ++k)
#pragma unroll
          for (int i = 0; i < NIT; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] += col[(i * V + j) * WG + k * TPR + t];
    }
  };
  if (!a.want) return;
  if (a.y) across(aw);
  if (a.y && LAYER) across(ab);
  if (a.pre) across(cw);
  if (a.pre && LAYER) across(cb);
  if (threadIdx.x >= TPR) return;
  float* out = a.part + (long long)blockIdx.x * 5 * C;
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    float sw[V], sb[V], w2[V], b2[V];
    take(sw, aw, kAw, i);
    take(w2, cw, kCw, i);
    if (LAYER) {
      take(sb, ab, kAb, i);
      take(b2, cb, kCb, i);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (i * TPR + t) * V + j;
      if (c >= C) continue;
      const float gate = a.gate && !per_row ? (float)gv[i].e[j] : 1.f;
      if (a.want & 1) out[c] = a.scale * gate * sw[j];
      if (LAYER && (a.want & 2)) out[C + c] = a.scale * gate * sb[j];
      if (a.want & 4) out[2 * C + c] = w2[j];
      if (LAYER && (a.want & 8)) out[3 * C + c] = b2[j];
      if (a.want & 16) {
        const float w = a.pw ? (float)pw[i].e[j] : 1.f;
        out[4 * C + c] = a.scale * (a.post ? fmaf(sw[j], w, LAYER && a.pb ? (float)pb[i].e[j] * sb[j] : 0.f) : sw[j]);
      }
    }
  }
}

// Adds the partial rows of a column: W columns x 1024 / W shares of the chunks per workgroup; blockIdx.y = quantity (0..3) or 4 + gate row
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* part, long long chunks, int cpg, int C, int W, void* o0, void* o1, void* o2, void* o3,
                                                          void* o4) {
  __shared__ float s[1024];
  const int k = blockIdx.y < 4 ? blockIdx.y : 4;
  void* o = k == 0 ? o0 : k == 1 ? o1 : k == 2 ? o2 : k == 3 ? o3 : o4;
  if (!o) return;
  const long long gr = (long long)blockIdx.y - 4, lo = k < 4 ? 0 : gr * cpg, n = k < 4 ? chunks : cpg;
  const int x = threadIdx.x % W, c = blockIdx.x * W + x, share = threadIdx.x / W, shares = 1024 / W;
  float v = 0.f;
  if (c < C) {
    const float* p = part + ((lo * 5 + k) * C + c);
    float u[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    long long i = share;
    for (; i + 7 * shares < n; i += 8 * shares)
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += p[(i + j * shares) * 5 * C];
    for (int j = 0; i < n; i += shares, ++j) u[j & 7] += p[i * 5 * C];
    v = ((u[0] + u[1]) + (u[2] + u[3])) + ((u[4] + u[5]) + (u[6] + u[7]));
  }
  s[threadIdx.x] = v;
  for (int d = shares / 2; d >= 1; d /= 2) {
    __syncthreads();
    if (share < d) s[threadIdx.x] += s[threadIdx.x + d * W];
  }
  if (share == 0 && c < C) ((T*)o)[(k < 4 ? 0 : gr * C) + c] = (T)s[x];
}

constexpr long long kMostGates = 60000;            // shared gate rows whose gradients are formed (a workgroup row of the column sums each)

// chunks: as many workgroups as the chip holds at a time (three per CU, two for the layer norm's registers), none across a gate row that is kept for a chunk
static long long cut_rows(NormArgs& a, int rpb) {
  a.span = a.gate && !a.each ? a.rpg : a.rows;
  const long long gates = a.rows / a.span;         // (check_norm: rows divide into gate rows)
  const long long want = a.layer ? 512 : 768;
  long long cpg = (want + gates - 1) / gates;
  const long long most = (a.span + rpb - 1) / rpb;
  if (cpg > most) cpg = most;
  a.rpc = (a.span + cpg - 1) / cpg;
  a.rpc = (a.rpc + rpb - 1) / rpb * rpb;
  a.cpg = (int)((a.span + a.rpc - 1) / a.rpc);
  return gates * a.cpg;
}

struct Shape { int v, tpr, nit; };

static Shape shape_for(int C, int dtype, bool vec) {
  const int v = vec ? (dtype == PGRF_DTYPE_F32 ? 4 : 8) : 1;
  const int n = (C + 7) / 8;                         // threads of eight values
  if (v == 4 && C <= 16) return {4, 4, 1};
  if (v == 1 && C <= 16) return {1, 16, 1};
  int tpr = n <= 4 ? 4 : n <= 16 ? 16 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : n <= 512 ? 512 : 1024;
  return {v, tpr, 8 / v};
}

static bool rows_vectorise(int C, int dtype, const void* const* ps, int n) {
  if (C % (dtype == PGRF_DTYPE_F32 ? 4 : 8)) return false;
  for (int i = 0; i < n; ++i)
    if (ps[i] && !aligned16(ps[i])) return false;
  return true;
}

template <typename T, int V, int TPR, int NIT>
static void run_norm(const NormArgs& a, long long chunks, bool bwd, hipStream_t s) {
  constexpr int WG = TPR > 256 ? TPR : 256;
  if (bwd) {
    if (a.layer) hipLaunchKernelGGL((block_norm_bwd_kernel<T, V, TPR, NIT, true>), dim3((unsigned)chunks), dim3(WG), 0, s, a);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<T, V, TPR, NIT, false>), dim3((unsigned)chunks), dim3(WG), 0, s, a);
    return;
  }
  const long long need = (a.rows + WG / TPR - 1) / (WG / TPR), most = 8 * 256 * 256 / WG;
  hipLaunchKernelGGL((block_norm_kernel<T, V, TPR, NIT>), dim3((unsigned)(need < most ? need : most)), dim3(WG), 0, s, a);
}

template <typename T>
static void pick_norm(const NormArgs& a, const Shape& h, long long chunks, bool bwd, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
#define PGRF_NORM(VV, TT, NN) \
  if (h.v == VV && h.tpr == TT && h.nit == NN) return run_norm<T, VV, TT, NN>(a, chunks, bwd, s)
#define PGRF_NORMS(VV) \
  PGRF_NORM(VV, 4, 8 / VV); PGRF_NORM(VV, 16, 8 / VV); PGRF_NORM(VV, 64, 8 / VV); PGRF_NORM(VV, 128, 8 / VV); PGRF_NORM(VV, 256, 8 / VV); \
  PGRF_NORM(VV, 512, 8 / VV); PGRF_NORM(VV, 1024, 8 / VV)
  PGRF_NORMS(V);
  PGRF_NORMS(1);
  if constexpr (V == 4) { PGRF_NORM(4, 4, 1); }
  PGRF_NORM(1, 16, 1);
#undef PGRF_NORMS
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

static NormArgs args_of(const PgrfBlockNorm* p) {
  NormArgs a = {};
  a.post = (p->flags & PGRF_NORM_POST) ? 1 : 0; a.pre = (p->flags & PGRF_NORM_PRE) ? 1 : 0; a.layer = (p->flags & PGRF_NORM_LAYER) ? 1 : 0;
  a.x = p->x; a.y = p->y; a.gate = p->gate; a.rpg = p->gate ? p->rows_per_gate : (p->rows ? p->rows : 1);
  a.pw = a.post ? p->post_w : nullptr; a.pb = a.post && a.layer ? p->post_b : nullptr; a.qw = a.pre ? p->pre_w : nullptr;
  a.stats = p->stats; a.rows = p->rows; a.C = p->C; a.scale = p->scale;
  return a;
}

}  // namespace tok
}  // namespace pgrf

using namespace pgrf;
using namespace pgrf::tok;

extern "C" {

int pgrf_block_norm(const PgrfBlockNorm* p, void* stream) {
  const char* who = "pgrf_block_norm";
  if (!p) return set_error(PGRF_ERR_ARG, "%s: null arguments", who);
  int rc = check_norm(who, p->dtype, p->rows, p->C, p->flags, p->rows_per_gate, p->y, p->gate);
  if (rc) return rc;
  if (p->rows == 0) return PGRF_OK;
  if (!p->x || (p->y && !p->x_out) || ((p->flags & PGRF_NORM_PRE) && !p->z_out)) return set_error(PGRF_ERR_ARG, "%s: null x / x_out / z_out", who);
  if (p->stats && !aligned16(p->stats)) return set_error(PGRF_ERR_ARG, "%s: stats must be 16-byte aligned", who);
  NormArgs a = args_of(p);
  a.qb = a.pre && a.layer ? p->pre_b : nullptr;
  a.xo = p->y ? p->x_out : nullptr; a.z = p->z_out; a.eps = p->eps;
  const void* ps[] = {a.x, a.y, a.gate, a.pw, a.pb, a.qw, a.qb, a.xo, a.pre ? a.z : nullptr};
  dispatch_norm(a, p->dtype, shape_for(p->C, p->dtype, rows_vectorise(p->C, p->dtype, ps, 9)), 0, false, (hipStream_t)stream);
  PGRF_TOK_LAUNCHED(who);
  return PGRF_OK;
}

size_t pgrf_block_norm_backward_workspace_bytes(long long rows, int C, long long rows_per_gate) {
  if (rows < 1 || C < 1 || rows_per_gate < 1) return 16;
  // an upper bound of cut_rows' chunks: 768, plus one for each gate row that is kept for a chunk
  const long long gates = rows_per_gate > 1 ? (rows + rows_per_gate - 1) / rows_per_gate : 1;
  return (size_t)(768 + (gates > kMostGates ? 1 : gates)) * 5 * (size_t)C * sizeof(float);
}

int pgrf_block_norm_backward(const PgrfBlockNorm* p, void* stream) {
  const char* who = "pgrf_block_norm_backward";
  if (!p) return set_error(PGRF_ERR_ARG, "%s: null arguments", who);
  int rc = check_norm(who, p->dtype, p->rows, p->C, p->flags, p->rows_per_gate, p->y, p->gate);
  if (rc) return rc;
  if (p->dgate && !p->gate) return set_error(PGRF_ERR_ARG, "%s: dgate without gate", who);
  NormArgs a = args_of(p);
  if (p->rows && (!p->stats || !p->x)) return set_error(PGRF_ERR_ARG, "%s: null stats / x", who);
  if (p->rows && !aligned16(p->stats)) return set_error(PGRF_ERR_ARG, "%s: stats must be 16-byte aligned", who);
  a.dxo = p->dx_out; a.dz = a.pre ? p->dz : nullptr; a.dx = p->dx; a.dy = p->y ? p->dy : nullptr;
  const bool per_row = p->gate && p->rows_per_gate == 1;
  a.dgate = per_row ? p->dgate : nullptr;
  a.part = (float*)p->workspace;
  a.want = (a.post && p->dpost_w ? 1 : 0) | (a.post && a.layer && p->dpost_b ? 2 : 0) | (a.pre && p->dpre_w ? 4 : 0) | (a.pre && a.layer && p->dpre_b ? 8 : 0) |
           (p->dgate && !per_row ? 16 : 0);
  const void* ps[] = {a.x, a.y, a.gate, a.pw, a.pb, a.qw, a.dxo, a.dz, a.dx, a.dy, a.dgate};
  const int C = p->C;
  const Shape h = shape_for(C, p->dtype, rows_vectorise(C, p->dtype, ps, 11));
  long long chunks = 0;
  a.cpg = 1;
  const long long gates = (a.want & 16) && p->rows ? p->rows / p->rows_per_gate : 0;
  if (gates > kMostGates) return set_error(PGRF_ERR_UNSUPPORTED, "%s: gradients of %lld gate rows (at most %lld, or one for each row)", who, gates, kMostGates);
  a.each = per_row || (p->gate && p->rows / p->rows_per_gate > kMostGates) ? 1 : 0;
  if (p->rows) {
    chunks = cut_rows(a, h.tpr > 256 ? 1 : 256 / h.tpr);
    const size_t need = (size_t)chunks * 5 * C * sizeof(float);
    if (a.want && (!p->workspace || p->workspace_bytes < need)) return set_error(PGRF_ERR_ARG, "%s: workspace too small (%zu < %zu bytes)", who, p->workspace_bytes, need);
    dispatch_norm(a, p->dtype, h, chunks, true, (hipStream_t)stream);
    PGRF_TOK_LAUNCHED(who);
  }
  if (a.want) {
    int W = 64;
    while (W > 4 && W / 2 >= C) W /= 2;
    const dim3 grid((C + W - 1) / W, 4 + (unsigned)gates);
    void *o0 = a.want & 1 ? p->dpost_w : nullptr, *o1 = a.want & 2 ? p->dpost_b : nullptr, *o2 = a.want & 4 ? p->dpre_w : nullptr,
         *o3 = a.want & 8 ? p->dpre_b : nullptr, *o4 = a.want & 16 ? p->dgate : nullptr;
#define PGRF_COLS(T) hipLaunchKernelGGL(column_sum_kernel<T>, grid, dim3(1024), 0, (hipStream_t)stream, a.part, chunks, a.cpg, C, W, o0, o1, o2, o3, o4)
    if (p->dtype == PGRF_DTYPE_F32) PGRF_COLS(float);
    else if (p->dtype == PGRF_DTYPE_BF16) PGRF_COLS(bf16);
    else PGRF_COLS(f16);
#undef PGRF_COLS
    PGRF_TOK_LAUNCHED(who);
  }
  return PGRF_OK;
}

}  // extern "C"
