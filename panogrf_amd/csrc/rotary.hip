// Rotary positions: the pair i of a head's first `rot` channels is turned by the angle  position * f_i,  f_i = base^(-2i/rot), scaled for long
// contexts; the gradient is the turn by the opposite angle, so one kernel serves both directions.
//   half layout: pair i = channels (i, i + rot/2);  interleaved: channels (2i, 2i + 1);  channels behind `rot` are copied
//
// The angle of a far position needs more than float: f_i / 2 pi (revolutions by position) comes from the host in double, the product is taken and
// reduced to a fraction of a revolution in double, and only the fraction goes to the float sine and cosine.  A workgroup forms them once for its
// tokens in LDS and turns the query and key heads of those tokens with them; what is left is one read and one write of every value, so memory
// bounds it (bf16, 32768 tokens x 32 heads x 64: 58 us, 4.6 TB/s where a copy has 5.2; float, 131072 x 8 x 32: 54 us, 4.9).
#include <cmath>

#include "pgrf_experiments.h"
#include "token_common.h"

namespace pgrf {
namespace tok {

constexpr int kMaxPairs = PGRF_ROTARY_MAX_DIM / 2, kMaxTile = 64;

struct Strided { const void* in; void* out; long long sb, sn, sh; int heads; };   // in: [B,N,heads,D] by strides; out: contiguous

struct RotaryArgs {
  Strided x[2];
  const void* pos;
  long long pos_b;               // stride of the positions' batch axis (0: shared)
  int pos_kind, B, N, D, rot, tile, interleaved;
  float sign, magnitude, inv_items, inv_per_head;
  int items;                     // work items of a token
  int per_head;                  // work items of a head
  double rev[kMaxPairs];         // revolutions by position
};

// n / d for 0 <= n < 2^21 with inv = 1.f / d: n + 0.5 lies at least 0.5 from every multiple of d, which the rounding of the product cannot bridge
__device__ __forceinline__ int quick_div(int n, float inv) { return (int)(((float)n + 0.5f) * inv); }

enum { kPairs = 0, kHalves = 1, kAnyHalves = 2 };

// An item is what a thread moves at a time: V neighbouring channels (interleaved pairs, or halves that vectors straddle), or two vectors - V pairs, or what
// is copied behind them.  A thread has two items on their way at once.
template <typename T, int V, int HOW>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 turn[];                   // [tile][rot/2]: cos, sin
  __shared__ long long from[2][kMaxTile];            // where a token's query and key heads start
  const int half = a.rot >> 1;
  const long long tokens = (long long)a.B * a.N, t0 = (long long)blockIdx.x * a.tile;
  const int here = tokens - t0 < a.tile ? (int)(tokens - t0) : a.tile;
  const long long b0 = t0 / a.N, n0 = t0 - b0 * a.N;
  auto place = [&](int k, long long& b, long long& n) {   // batch entry and place of the tile's token k
    b = b0;
    n = n0 + k;
    if (n >= a.N) {
      const unsigned more = (unsigned)n / (unsigned)a.N;   // (n < 2^31 + a tile)
      b += more;
      n -= (long long)more * a.N;
    }
  };
  for (int i = threadIdx.x; i < here * half; i += 256) {
    const int k = i / half, pair = i - k * half;
    long long b, n;
    place(k, b, n);
    const long long at = b * a.pos_b + n;
    const double p = a.pos_kind == 0 ? (double)((const int*)a.pos)[at] : a.pos_kind == 1 ? (double)((const long long*)a.pos)[at]
                   : a.pos_kind == 2 ? (double)((const float*)a.pos)[at] : ((const double*)a.pos)[at];
    const double r = p * a.rev[pair];
    const float f = 2.f * (float)(r - rint(r));
    float s, c;
    sincospif(f, &s, &c);
    turn[i] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
  if ((int)threadIdx.x < 2 * here) {
    const int k = threadIdx.x >> 1, w = threadIdx.x & 1;
    long long b, n;
    place(k, b, n);
    from[w][k] = b * a.x[w].sb + n * a.x[w].sn;
  }
  __syncthreads();
  const int total = here * a.items, np = half / V;
  struct Item { Vec<T, V> u, w; T* out; const T* in; const float2* cs; int j; bool has_w; };
  auto bring = [&](Item& m, int it) {
    const int k = quick_div(it, a.inv_items), rem = it - k * a.items;
    int head = quick_div(rem, a.inv_per_head);
    m.j = rem - head * a.per_head;
    const int which = head >= a.x[0].heads ? 1 : 0;
    if (which) head -= a.x[0].heads;
    const long long sh = which ? a.x[1].sh : a.x[0].sh;
    const int heads = which ? a.x[1].heads : a.x[0].heads;
    m.in = (const T*)(which ? a.x[1].in : a.x[0].in) + from[which][k] + head * sh;
    m.out = (T*)(which ? a.x[1].out : a.x[0].out) + ((t0 + k) * heads + head) * a.D;
    m.cs = turn + k * half;
    if constexpr (HOW == kHalves) {
      const bool pair = m.j < np;
      const int c0 = pair ? m.j * V : a.rot + 2 * (m.j - np) * V, c1 = pair ? c0 + half : c0 + V;
      m.has_w = c1 < a.D;
      m.u = load_vec<T, V>(m.in + c0);
      if (m.has_w) m.w = load_vec<T, V>(m.in + c1);
    } else {
      m.u = load_vec<T, V>(m.in + m.j * V);
    }
  };
  auto finish = [&](Item& m) {
    if constexpr (HOW == kHalves) {
      const bool pair = m.j < np;
      const int c0 = pair ? m.j * V : a.rot + 2 * (m.j - np) * V, c1 = pair ? c0 + half : c0 + V;
      if (pair) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 q = m.cs[c0 + e];
          const float p = (float)m.u.e[e], r = (float)m.w.e[e];
          m.u.e[e] = (T)(p * q.x - r * q.y);
          m.w.e[e] = (T)(r * q.x + p * q.y);
        }
      }
      store_vec<T, V>(m.out + c0, m.u);
      if (m.has_w) store_vec<T, V>(m.out + c1, m.w);
    } else {
      const int c0 = m.j * V;
      Vec<T, V> o = m.u;
      if constexpr (HOW == kPairs && V == 1) {
        if (c0 < a.rot) {
          const float2 q = m.cs[c0 >> 1];
          const float p = (float)m.u.e[0], r = (float)m.in[c0 ^ 1];
          o.e[0] = (T)((c0 & 1) ? p * q.x + r * q.y : p * q.x - r * q.y);
        }
      } else if constexpr (HOW == kPairs) {
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2)
          if (c0 + e < a.rot) {
            const float2 q = m.cs[(c0 + e) >> 1];
            const float p = (float)m.u.e[e], r = (float)m.u.e[e + 1];
            o.e[e] = (T)(p * q.x - r * q.y);
            o.e[e + 1] = (T)(r * q.x + p * q.y);
          }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = c0 + e;
          if (c < a.rot) {
            const bool low = c < half;
            const float2 q = m.cs[low ? c : c - half];
            const float p = (float)m.u.e[e], r = (float)m.in[low ? c + half : c - half];
            o.e[e] = (T)(low ? p * q.x - r * q.y : p * q.x + r * q.y);
          }
        }
      }
      store_vec<T, V>(m.out + c0, o);
    }
  };
  for (int it = threadIdx.x; it < total; it += 512) {
    Item m0, m1;
    bring(m0, it);
    const bool two = it + 256 < total;
    if (two) bring(m1, it + 256);
    finish(m0);
    if (two) finish(m1);
  }
}

template <typename T>
static void launch_rotary(const RotaryArgs& a, bool vec, dim3 grid, size_t lds, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (a.interleaved) {
    if (vec) hipLaunchKernelGGL((rotary_kernel<T, V, kPairs>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((rotary_kernel<T, 1, kPairs>), grid, dim3(256), lds, s, a);
  } else if (vec && (a.rot / 2) % V == 0) {
    hipLaunchKernelGGL((rotary_kernel<T, V, kHalves>), grid, dim3(256), lds, s, a);
  } else if (vec) {
    hipLaunchKernelGGL((rotary_kernel<T, V, kAnyHalves>), grid, dim3(256), lds, s, a);
  } else {
    hipLaunchKernelGGL((rotary_kernel<T, 1, kAnyHalves>), grid, dim3(256), lds, s, a);
  }
}

}  // namespace tok
}  // namespace pgrf

using namespace pgrf;
using namespace pgrf::tok;

extern "C" int pgrf_rotary(const PgrfRotary* p, void* stream) {
  const char* who = "pgrf_rotary";
  if (!p) return set_error(PGRF_ERR_ARG, "%s: null arguments", who);
  const int dtype = p->dtype, B = p->B, N = p->N, D = p->D, q_heads = p->q_heads, k_heads = p->k_heads, rotary_dim = p->rotary_dim, scaling = p->scaling;
  const double base = p->base, factor = p->factor, trained_length = p->trained_length, low = p->low, high = p->high;
  const void *q = p->q, *k = p->k;
  void *q_out = p->q_out, *k_out = p->k_out;
  const long long q_sb = p->q_sb, q_sn = p->q_sn, q_sh = p->q_sh, k_sb = p->k_sb, k_sn = p->k_sn, k_sh = p->k_sh;
  if (!dtype_ok(dtype)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: dtype %d (PGRF_DTYPE_F32 | BF16 | F16)", who, dtype);
  if (B < 0 || N < 0 || q_heads < 1 || k_heads < 0 || D < 2) return set_error(PGRF_ERR_ARG, "%s: bad sizes B=%d N=%d heads=%d,%d D=%d", who, B, N, q_heads, k_heads, D);
  if (rotary_dim < 2 || (rotary_dim & 1) || rotary_dim > D || rotary_dim > PGRF_ROTARY_MAX_DIM)
    return set_error(PGRF_ERR_UNSUPPORTED, "%s: rotary_dim=%d (even, at most the head's %d channels and %d)", who, rotary_dim, D, PGRF_ROTARY_MAX_DIM);
  if ((long long)(q_heads + (long long)k_heads) * D > (1 << 20)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: over 2^20 channels by token", who);
  if (p->position_type < 0 || p->position_type > 3) return set_error(PGRF_ERR_ARG, "%s: position_type %d", who, p->position_type);
  if (!(base > 0) || !std::isfinite(base)) return set_error(PGRF_ERR_ARG, "%s: base must be positive", who);
  if (scaling < PGRF_ROTARY_PLAIN || scaling > PGRF_ROTARY_PARTS) return set_error(PGRF_ERR_ARG, "%s: scaling %d", who, scaling);
  if (scaling != PGRF_ROTARY_PLAIN && !(factor > 0 && std::isfinite(factor))) return set_error(PGRF_ERR_ARG, "%s: factor must be positive", who);
  if (scaling == PGRF_ROTARY_NTK && rotary_dim < 4) return set_error(PGRF_ERR_UNSUPPORTED, "%s: this scaling needs rotary_dim of 4 at least", who);
  if (scaling == PGRF_ROTARY_PARTS && !(trained_length > 0 && high > low)) return set_error(PGRF_ERR_ARG, "%s: scaling by parts needs trained_length > 0 and high > low", who);
  if ((long long)B * N == 0) return PGRF_OK;
  if (!q || !q_out || !p->positions || (k_heads && (!k || !k_out))) return set_error(PGRF_ERR_ARG, "%s: null pointer", who);
  RotaryArgs a = {};
  a.x[0] = {q, q_out, q_sb, q_sn, q_sh, q_heads};
  a.x[1] = {k, k_out, k_sb, k_sn, k_sh, k_heads};
  a.pos = p->positions; a.pos_b = p->pos_sb; a.pos_kind = p->position_type;
  a.B = B; a.N = N; a.D = D; a.rot = rotary_dim; a.interleaved = p->interleaved ? 1 : 0;
  a.sign = p->backward ? -1.f : 1.f; a.magnitude = p->magnitude;
  const double pi2 = 6.283185307179586476925286766559, bs = scaling == PGRF_ROTARY_NTK ? base * std::pow(factor, rotary_dim / (rotary_dim - 2.0)) : base;
  const double step = -2.0 * std::log2(bs) / rotary_dim;
  for (int i = 0; i < rotary_dim / 2; ++i) {
    double f = std::exp2(step * i);
    if (scaling == PGRF_ROTARY_LINEAR) f /= factor;
    if (scaling == PGRF_ROTARY_PARTS) {
      double keep = (trained_length * f / pi2 - low) / (high - low);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      f = f * (keep + (1 - keep) / factor);
    }
    a.rev[i] = f / pi2;
  }
  const int V = 16 / (int)dtype_bytes(dtype);
  bool vec = D % V == 0 && aligned16(q) && aligned16(q_out) && !((q_sb | q_sn | q_sh) % V);
  if (k_heads) vec = vec && aligned16(k) && aligned16(k_out) && !((k_sb | k_sn | k_sh) % V);
  const int step_v = vec ? V : 1;
  const bool halves = !p->interleaved && vec && (rotary_dim / 2) % V == 0;
  a.per_head = halves ? rotary_dim / 2 / V + ((D - rotary_dim) / V + 1) / 2 : D / step_v;
  a.items = (q_heads + k_heads) * a.per_head;
  a.inv_items = 1.f / a.items;
  a.inv_per_head = 1.f / a.per_head;
  // Tokens of a workgroup: about eight items per thread, as long as over a thousand workgroups remain, and 32 KB of sines at most
  const long long tokens = (long long)B * N;
  long long tile = 2048 / a.items;
  if (tile > tokens / 1024) tile = tokens / 1024;
  if (tile > 4096 / (rotary_dim / 2)) tile = 4096 / (rotary_dim / 2);
  if (tile > kMaxTile) tile = kMaxTile;
  const long long least = tokens / 0xffffff + 1;    // a launch holds 2^32 - 1 threads, 256 a workgroup
  if (tile < least) tile = least;
  if (tile > kMaxTile || tile * a.items >= (1 << 21) || (tile > 1 && tile * (rotary_dim / 2) > 4096)) return set_error(PGRF_ERR_UNSUPPORTED, "%s: too many tokens", who);   // (2^21: quick_div)
  a.tile = (int)tile;
  const long long grid = (tokens + a.tile - 1) / a.tile;
  const size_t lds = (size_t)a.tile * (rotary_dim / 2) * sizeof(float2);
  if (dtype == PGRF_DTYPE_F32) launch_rotary<float>(a, vec, dim3((unsigned)grid), lds, (hipStream_t)stream);
  else if (dtype == PGRF_DTYPE_BF16) launch_rotary<bf16>(a, vec, dim3((unsigned)grid), lds, (hipStream_t)stream);
  else launch_rotary<f16>(a, vec, dim3((unsigned)grid), lds, (hipStream_t)stream);
  PGRF_TOK_LAUNCHED(who);
  return PGRF_OK;
}
