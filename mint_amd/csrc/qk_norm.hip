// RMS norm of every query and key head with a learned gain, then rotation by position, forward and backward
// (definition: include/fact_hip.h, FactQkNorm).
//
// Forward   r = rsqrt(mean x^2 + eps), y = x r gamma, z = R(pos) y
// Backward  dy = R(pos)^T dz, dgamma = sum dy x r, dx = r (gamma dy - x r mean(gamma dy x r))
// Both read each value once and write each result once.  In fp32 the rate of the copy they amount to bounds them: B 8, n 1440,
// 24 heads of 128 takes 54 us forward (5.2 TB/s) and 91 + 5 backward (4.6 TB/s).  In bf16, B 16, n 360, 20 heads of 80, which caches
// hold, 12 and 17 + 4, where the copy would take 7 and 11: 10 of a group's 16 lanes and 10 of a piece's 12 heads are in use, half of
// the lanes, by 8-byte loads.  One token of 32 sequences takes 4.  (Launches under the profiler.)  A head of dh
// values is held by dh / 8 lanes of a group of GL = 4, 8 or 16 (its row sums stay inside a 16-lane row); a lane holds 4 pairs
// of one rotation slot, so the partner of every value is in the same lane.  A wave takes heads of one token, of the queries or
// of the keys: the angles, reduced in double (a far position times a frequency loses whole turns in 32 bits), are computed once
// for all of them.
#include "rel_attention.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

namespace {

struct Side {  // queries or keys
  const void* x;        // the projections
  const void* e;        // backward: gradient of the outputs
  void* y;              // forward: outputs; backward: gradient of the projections
  const float* gamma;
  float* dgamma;
  int64_t xs[3], es[3], ys[3];
  int heads, pieces, blocks;  // pieces of a token's heads, workgroups
  unsigned units;             // tokens times pieces
};
struct NormP {
  Side side[2];
  const int32_t* positions;
  int64_t ps[2];
  double turn0, ratio[6];  // pair i turns by turn0 * (base^(-2 / rotary_dim))^i a position; ratio[k] = that power 2^k
  float* part;             // [workgroups][dh] gain gradients
  int n, dh, rotary_dim, interleaved, position0, accumulate;
  float eps;
};

// Heads in flight per lane group and piece.  Enough loads at once to cover the memory's latency, few enough registers for
// 4 waves per SIMD.
template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
  typedef f32x4 V;
  static constexpr int UF = 2, UB = 2;
};
template <>
struct Vec4<bf16_t> {
  typedef bf16x4 V;
  static constexpr int UF = 3, UB = 3;
};

template <typename T>
DEVINL typename Vec4<T>::V raw4(const T* p) { return *reinterpret_cast<const typename Vec4<T>::V*>(p); }
template <typename V>
DEVINL f32x4 wide(V v) { return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }
DEVINL f32x4 load4(const float* p) { return raw4(p); }
template <typename T>
DEVINL void store4(T* p, f32x4 v) {
  typename Vec4<T>::V o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  *reinterpret_cast<typename Vec4<T>::V*>(p) = o;
}
// sum over aligned groups of GL lanes by moves inside rows of 16
template <int CTRL>
DEVINL float plus_moved(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int GL>
DEVINL float group_sum(float v) {
  v = plus_moved<0xB1>(v);                        // lane ^ 1
  v = plus_moved<0x4E>(v);                        // lane ^ 2
  if constexpr (GL >= 8) v = plus_moved<0x141>(v);   // 7 - lane
  if constexpr (GL >= 16) v = plus_moved<0x140>(v);  // 15 - lane
  return v;
}

// a lane's place in its head: two runs of 4 values, at o0 and o1
struct Slot {
  int o0, o1;
  bool on, rot;
};
DEVINL Slot slot_of(const NormP& a, int s) {
  Slot r;
  r.on = s * 8 < a.dh;
  r.rot = s * 8 < a.rotary_dim;
  if (r.rot && !a.interleaved) {
    r.o0 = 4 * s;
    r.o1 = a.rotary_dim / 2 + 4 * s;
  } else {
    r.o0 = 8 * s;
    r.o1 = 8 * s + 4;
  }
  return r;
}
// a wave's lanes each take one pair of the token (there are at most 64) and hand the results to the lanes that turn them
DEVINL void angles(const NormP& p, int pos, int s, int lane, f32x4& co, f32x4& si) {
  double turn = p.turn0;
#pragma unroll
  for (int k = 0; k < 6; ++k) turn *= (lane >> k) & 1 ? p.ratio[k] : 1.0;
  double x = pos * turn;
  x -= rint(x);
  // (The rest, at most half a turn, in 32 bits: an angle is off by 2^-24 of up to pi, 2^-22.3.  fp32 results are 6.2e-8 off in
  // norm with it, and 5.8e-8 with cosines and sines of 64 bits.)
  float u, w;
  sincospif((float)(2.0 * x), &u, &w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int from = min(4 * s + i, 63);
    si[i] = __shfl(u, from, 64);
    co[i] = __shfl(w, from, 64);
  }
}
DEVINL int position(const NormP& p, int b, int t) {
  return p.positions ? p.positions[b * p.ps[0] + t * p.ps[1]] : p.position0 + t;
}
// (a, b) -> (a c - b s, b c + a s); the pairs are (a[i], b[i]) or neighbours in a, then in b
DEVINL void turn4(f32x4& a, f32x4& b, f32x4 c, f32x4 s, bool inter) {
  if (inter) {
    const f32x4 x = a, y = b;
    a = f32x4{x[0] * c[0] - x[1] * s[0], x[1] * c[0] + x[0] * s[0], x[2] * c[1] - x[3] * s[1], x[3] * c[1] + x[2] * s[1]};
    b = f32x4{y[0] * c[2] - y[1] * s[2], y[1] * c[2] + y[0] * s[2], y[2] * c[3] - y[3] * s[3], y[3] * c[3] + y[2] * s[3]};
  } else {
    const f32x4 x = a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = x[i] * c[i] - b[i] * s[i];
      b[i] = b[i] * c[i] + x[i] * s[i];
    }
  }
}

// a piece: up to NG * U heads of one token
struct Piece {
  int b, t, h;  // h: this lane group's first head, the others follow NG apart
};
DEVINL Piece piece_of(const NormP& p, const Side& d, unsigned unit, int rows, int gr) {
  const unsigned tok = unit / (unsigned)d.pieces;
  Piece c;
  c.h = (int)(unit - tok * d.pieces) * rows + gr;
  c.b = (int)(tok / (unsigned)p.n);
  c.t = (int)(tok - (unsigned)c.b * p.n);
  return c;
}

template <typename T, int GL>
__global__ __launch_bounds__(256, 4) void qk_norm_kernel(const NormP p) {
  constexpr int NG = 64 / GL, U = Vec4<T>::UF;
  const int lane = threadIdx.x & 63, s = lane % GL, gr = lane / GL;
  const bool isk = (int)blockIdx.x >= p.side[0].blocks;
  const Side& d = p.side[isk];
  const unsigned unit = (blockIdx.x - (isk ? p.side[0].blocks : 0)) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= d.units) return;
  const Piece c = piece_of(p, d, unit, NG * U, gr);
  const Slot sl = slot_of(p, s);
  typename Vec4<T>::V x[U][2] = {};
  const int pos = p.rotary_dim ? position(p, c.b, c.t) : 0;
  const T* in = (const T*)d.x + (c.b * d.xs[0] + c.t * d.xs[1]) + c.h * d.xs[2];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (sl.on && c.h + u * NG < d.heads) {
      x[u][0] = raw4(in + u * NG * d.xs[2] + sl.o0);
      x[u][1] = raw4(in + u * NG * d.xs[2] + sl.o1);
    }
  f32x4 co = {1.f, 1.f, 1.f, 1.f}, si = {0.f, 0.f, 0.f, 0.f}, ga[2];
  ga[0] = sl.on && d.gamma ? load4(d.gamma + sl.o0) : f32x4{1.f, 1.f, 1.f, 1.f};
  ga[1] = sl.on && d.gamma ? load4(d.gamma + sl.o1) : f32x4{1.f, 1.f, 1.f, 1.f};
  if (p.rotary_dim) angles(p, pos, s, lane, co, si);
  const float inv = 1.0f / p.dh;
  T* out = (T*)d.y + (c.b * d.ys[0] + c.t * d.ys[1]) + c.h * d.ys[2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    f32x4 y[2] = {wide(x[u][0]), wide(x[u][1])};
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += y[0][i] * y[0][i] + y[1][i] * y[1][i];
    const float r = rsqrtf(group_sum<GL>(ss) * inv + p.eps);
    if (!sl.on || c.h + u * NG >= d.heads) continue;
    y[0] = y[0] * r * ga[0];
    y[1] = y[1] * r * ga[1];
    if (sl.rot) turn4(y[0], y[1], co, si, p.interleaved != 0);
    store4(out + u * NG * d.ys[2] + sl.o0, y[0]);
    store4(out + u * NG * d.ys[2] + sl.o1, y[1]);
  }
}

template <typename T, int GL>
__global__ __launch_bounds__(512, 4) void qk_norm_bwd_kernel(const NormP p) {
  constexpr int NG = 64 / GL, U = Vec4<T>::UB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = lane % GL, gr = lane / GL;
  const bool isk = (int)blockIdx.x >= p.side[0].blocks;
  const Side& d = p.side[isk];
  const Slot sl = slot_of(p, s);
  f32x4 ga[2], acc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ga[i] = sl.on && d.gamma ? load4(d.gamma + (i ? sl.o1 : sl.o0)) : f32x4{1.f, 1.f, 1.f, 1.f};
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float inv = 1.0f / p.dh;
  for (unsigned unit = (blockIdx.x - (isk ? p.side[0].blocks : 0)) * 8 + wave; unit < d.units; unit += d.blocks * 8u) {
    const Piece c = piece_of(p, d, unit, NG * U, gr);
    typename Vec4<T>::V x[U][2] = {}, e[U][2] = {};
    const int pos = p.rotary_dim ? position(p, c.b, c.t) : 0;
    const T* in = (const T*)d.x + (c.b * d.xs[0] + c.t * d.xs[1]) + c.h * d.xs[2];
    const T* grad = (const T*)d.e + (c.b * d.es[0] + c.t * d.es[1]) + c.h * d.es[2];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (sl.on && c.h + u * NG < d.heads) {
        x[u][0] = raw4(in + u * NG * d.xs[2] + sl.o0);
        x[u][1] = raw4(in + u * NG * d.xs[2] + sl.o1);
        e[u][0] = raw4(grad + u * NG * d.es[2] + sl.o0);
        e[u][1] = raw4(grad + u * NG * d.es[2] + sl.o1);
      }
    f32x4 co = {1.f, 1.f, 1.f, 1.f}, si = {0.f, 0.f, 0.f, 0.f};
    if (p.rotary_dim) angles(p, pos, s, lane, co, si);
    T* out = (T*)d.y + (c.b * d.ys[0] + c.t * d.ys[1]) + c.h * d.ys[2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f32x4 y[2] = {wide(x[u][0]), wide(x[u][1])}, z[2] = {wide(e[u][0]), wide(e[u][1])};
      if (sl.rot) turn4(z[0], z[1], co, -si, p.interleaved != 0);
      float ss = 0.f, sd = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ss += y[i][j] * y[i][j];
          sd += y[i][j] * z[i][j] * ga[i][j];
        }
      const float r = rsqrtf(group_sum<GL>(ss) * inv + p.eps);
      const float k = group_sum<GL>(sd) * inv * r * r;
      if (!sl.on || c.h + u * NG >= d.heads) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        acc[i] += z[i] * (y[i] * r);
        store4(out + u * NG * d.ys[2] + (i ? sl.o1 : sl.o0), (z[i] * ga[i] - y[i] * k) * r);
      }
    }
  }
  // gain gradients: the groups of a wave, then the 8 waves, in one order
  __shared__ float red[8][128];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = GL; o < 64; o <<= 1) acc[i][j] += __shfl_xor(acc[i][j], o, 64);
  if (gr == 0 && sl.on) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) red[wave][(i ? sl.o1 : sl.o0) + j] = acc[i][j];
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i < p.dh)
    p.part[(size_t)blockIdx.x * p.dh + i] = ((red[0][i] + red[1][i]) + (red[2][i] + red[3][i])) +
                                            ((red[4][i] + red[5][i]) + (red[6][i] + red[7][i]));
}

// columns of a side's [blocks][dh] summed in row order: 8 columns a workgroup, 32 row groups
__global__ __launch_bounds__(256) void qk_norm_dgamma_kernel(const NormP p) {
  const int per = p.dh / 8, isk = (int)blockIdx.x >= per;
  const Side& d = p.side[isk];
  const int c = threadIdx.x & 7, r0 = threadIdx.x >> 3, i = ((int)blockIdx.x - isk * per) * 8 + c;
  const float* src = p.part + (isk ? (size_t)p.side[0].blocks * p.dh : 0) + i;
  __shared__ float red[32][9];
  float x = 0.f;
#pragma unroll 8
  for (int r = r0; r < d.blocks; r += 32) x += src[(size_t)r * p.dh];
  red[r0][c] = x;
  __syncthreads();
  if (r0 == 0 && d.dgamma) {
#pragma unroll
    for (int r = 1; r < 32; ++r) x += red[r][c];
    d.dgamma[i] = p.accumulate ? d.dgamma[i] + x : x;
  }
}

int lanes_of(const FactQkNorm& a) { return a.dh <= 32 ? 4 : a.dh <= 64 ? 8 : 16; }
int rows_of(const FactQkNorm& a, bool backward) {  // heads of a piece
  const int u = a.dtype ? (backward ? Vec4<float>::UB : Vec4<float>::UF) : (backward ? Vec4<bf16_t>::UB : Vec4<bf16_t>::UF);
  return 64 / lanes_of(a) * u;
}
// backward: together 2 workgroups of 8 waves for each of 256 CUs - as many as run at once, and few partial rows to add
void bwd_blocks(const FactQkNorm& a, int blocks[2]) {
  const int rows = rows_of(a, true);
  const long long tok = (long long)a.B * a.n, q = (a.H + rows - 1) / rows, k = (a.Hkv + rows - 1) / rows;
  const long long share = std::max(1ll, std::min(511ll, 512 * q / (q + k)));
  blocks[0] = (int)std::min(share, (tok * q + 7) / 8);
  blocks[1] = (int)std::min(512 - share, (tok * k + 7) / 8);
}

NormP params(const FactQkNorm& a, bool backward) {
  NormP p;
  memset(&p, 0, sizeof(p));
  const int rows = rows_of(a, backward);
  int blocks[2];
  bwd_blocks(a, blocks);
  auto fill = [&](Side& d, const void* x, const int64_t* xs, const void* e, const int64_t* es, void* y, const int64_t* ys, int heads) {
    d.x = x; d.e = e; d.y = y; d.heads = heads;
    for (int i = 0; i < 3; ++i) { d.xs[i] = xs[i]; d.es[i] = es[i]; d.ys[i] = ys[i]; }
    d.pieces = (heads + rows - 1) / rows;
    d.units = (unsigned)((long long)a.B * a.n * d.pieces);
  };
  fill(p.side[0], a.q, a.q_stride, a.dq_out, a.dq_out_stride, backward ? a.dq : a.q_out, backward ? a.dq_stride : a.q_out_stride, a.H);
  fill(p.side[1], a.k, a.k_stride, a.dk_out, a.dk_out_stride, backward ? a.dk : a.k_out, backward ? a.dk_stride : a.k_out_stride, a.Hkv);
  p.side[0].gamma = a.q_gamma; p.side[0].dgamma = a.dq_gamma;
  p.side[1].gamma = a.k_gamma; p.side[1].dgamma = a.dk_gamma;
  for (int i = 0; i < 2; ++i) p.side[i].blocks = backward ? blocks[i] : (int)((p.side[i].units + 3ll) / 4);
  p.positions = a.positions; p.ps[0] = a.position_stride[0]; p.ps[1] = a.position_stride[1];
  p.n = a.n; p.dh = a.dh; p.rotary_dim = a.rotary_dim; p.interleaved = a.interleaved; p.position0 = a.position0;
  p.accumulate = a.dgamma_accumulate; p.eps = a.eps;
  if (a.rotary_dim) {
    p.turn0 = 1.0 / 6.283185307179586476925286766559;
    for (int k = 0; k < 6; ++k) p.ratio[k] = std::pow(a.base, -2.0 * (1 << k) / a.rotary_dim);
  }
  return p;
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : -100; }

template <typename T, int GL>
int run(const FactQkNorm& a, bool backward, void* ws, hipStream_t s) {
  NormP p = params(a, backward);
  const unsigned grid = p.side[0].blocks + p.side[1].blocks;
  if (!backward) {
    FACT_LAUNCH((qk_norm_kernel<T, GL>), dim3(grid), dim3(256), 0, s, p);
    return launched();
  }
  p.part = (float*)ws;
  FACT_LAUNCH((qk_norm_bwd_kernel<T, GL>), dim3(grid), dim3(512), 0, s, p);
  if (a.dq_gamma || a.dk_gamma) FACT_LAUNCH(qk_norm_dgamma_kernel, dim3(2 * a.dh / 8), dim3(256), 0, s, p);
  return launched();
}
template <typename T>
int run(const FactQkNorm& a, bool backward, void* ws, hipStream_t s) {
  switch (lanes_of(a)) {
    case 4: return run<T, 4>(a, backward, ws, s);
    case 8: return run<T, 8>(a, backward, ws, s);
  }
  return run<T, 16>(a, backward, ws, s);
}

}  // namespace

int qk_norm_check(const FactQkNorm& a, bool backward, const char** why) {
  auto bad = [&](int rc, const char* w) { *why = w; return rc; };
  if (a.B <= 0 || a.n <= 0 || a.H <= 0 || a.Hkv <= 0) return bad(-1, "B, n, H and Hkv must be positive");
  // (pieces have at least 8 heads and workgroups 4 pieces; a launch has fewer than 2^32 threads, 256 a workgroup)
  if ((long long)a.H + a.Hkv > 65536 || (long long)a.B * a.n > 1 << 26 ||
      (long long)a.B * a.n * ((a.H + 7) / 8 + (a.Hkv + 7) / 8) > (1 << 26) - 8)
    return bad(-1, "too many tokens or heads");
  if (a.dh < 8 || a.dh > 128 || a.dh % 8) return bad(-3, "unsupported head dim (a multiple of 8 up to 128)");
  if (a.rotary_dim < 0 || a.rotary_dim > a.dh || a.rotary_dim % 8) return bad(-1, "rotary_dim must be a multiple of 8 up to dh");
  if (a.dtype != 0 && a.dtype != 1) return bad(-1, "dtype must be 0 (bf16) or 1 (fp32)");
  if (!a.positions && (long long)a.position0 + a.n - 1 > INT_MAX) return bad(-1, "the last token's position must fit 32 bits");
  if (!(a.eps >= 0.f) || !(a.eps < 3.0e38f)) return bad(-1, "eps must be finite and not negative");
  if (a.rotary_dim && !(a.base > 0.0 && a.base < 1e300)) return bad(-1, "base must be positive and finite");
  struct T { const void* p; const int64_t* st; int heads; bool out; };
  const T fwd[] = {{a.q, a.q_stride, a.H, false}, {a.k, a.k_stride, a.Hkv, false}, {a.q_out, a.q_out_stride, a.H, true},
                   {a.k_out, a.k_out_stride, a.Hkv, true}};
  const T bwd[] = {{a.q, a.q_stride, a.H, false}, {a.k, a.k_stride, a.Hkv, false}, {a.dq_out, a.dq_out_stride, a.H, false},
                   {a.dk_out, a.dk_out_stride, a.Hkv, false}, {a.dq, a.dq_stride, a.H, true}, {a.dk, a.dk_stride, a.Hkv, true}};
  const T* t = backward ? bwd : fwd;
  for (int i = 0; i < (backward ? 6 : 4); ++i) {
    if (!t[i].p) return bad(-1, "null tensor");
    if ((uintptr_t)t[i].p & 15) return bad(-1, "tensors must be 16-byte aligned");
    const int n[3] = {a.B, a.n, t[i].heads};
    for (int k = 0; k < 3; ++k) {
      if (t[i].st[k] & 7) return bad(-1, "strides must be multiples of 8 elements");
      if (t[i].out && t[i].st[k] == 0 && n[k] > 1) return bad(-1, "an output must not be broadcast");
    }
  }
  if (((uintptr_t)a.q_gamma | (uintptr_t)a.k_gamma) & 15) return bad(-1, "tensors must be 16-byte aligned");
  // Queries and keys are different workgroups of one launch, and a workgroup reads a value right before it writes the result in
  // its place: an output may stand where its own side's input does, value by value, and nowhere else.
  for (int i = 0; i < (backward ? 6 : 4); ++i)
    for (int k = 0; k < i; ++k) {
      if (t[i].p != t[k].p || !(t[i].out || t[k].out)) continue;
      const int n[3] = {a.B, a.n, t[i].heads};
      bool place = (i & 1) == (k & 1);  // (both lists alternate queries and keys)
      for (int j = 0; j < 3; ++j) place = place && (n[j] == 1 || t[i].st[j] == t[k].st[j]);
      if (!place) return bad(-1, "an output must not be another tensor (but its own input, with the same strides)");
    }
  if (backward) {
    const void* gains[] = {a.dq_gamma, a.dk_gamma};
    for (int i = 0; i < 2; ++i) {
      if (!gains[i]) continue;
      for (const void* x : {(const void*)a.q_gamma, (const void*)a.k_gamma, (const void*)a.positions, gains[1 - i]})
        if (gains[i] == x) return bad(-1, "an output must not be another tensor");
      for (const T& x : bwd)
        if (gains[i] == x.p) return bad(-1, "an output must not be another tensor");
    }
  }
  return 0;
}

size_t qk_norm_ws(const FactQkNorm& a, bool backward) { return backward ? (size_t)512 * a.dh * 4 : 0; }

int launch_qk_norm_fwd(const FactQkNorm& a, hipStream_t s) {
  return a.dtype ? run<float>(a, false, nullptr, s) : run<bf16_t>(a, false, nullptr, s);
}
int launch_qk_norm_bwd(const FactQkNorm& a, void* ws, hipStream_t s) {
  return a.dtype ? run<float>(a, true, ws, s) : run<bf16_t>(a, true, ws, s);
}
