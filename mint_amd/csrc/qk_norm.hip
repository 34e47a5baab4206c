// RMS norm of every query and key head with a learned gain, then rotation by position, forward and backward
// (definition: include/fact_hip.h, FactQkNorm).
//
// Forward   r = rsqrt(mean x^2 + eps), y = x r gamma, z = R(pos) y
// Backward  dy = R(pos)^T dz, dgamma = sum dy x r, dx = r (gamma dy - x r mean(gamma dy x r))
// Both read each value once and write each result once, so the rate of the copy they amount to bounds them.  A head of dh
// values is held by dh / 8 lanes of a group of GL = 4, 8 or 16 (its row sums stay inside a 16-lane row); a lane holds 4 pairs
// of one rotation slot, so the partner of every value is in the same lane.  A wave takes all heads of one token: the angles,
// reduced in double (a far position times a frequency loses whole turns in 32 bits), are computed once for all of them.
#include "rel_attention.h"

#include <climits>
#include <cmath>
#include <cstring>

namespace {

struct NormP {
  FactQkNorm a;
  double turn[64];  // frequency of pair i in turns per position
  float* part;      // [workgroups][2][dh] gain gradients
  long long tokens;
};

template <typename T>
struct Vec4;
template <>
struct Vec4<float> { typedef f32x4 V; };
template <>
struct Vec4<bf16_t> { typedef bf16x4 V; };

template <typename T>
DEVINL f32x4 load4(const T* p) {
  const typename Vec4<T>::V v = *reinterpret_cast<const typename Vec4<T>::V*>(p);
  return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <typename T>
DEVINL void store4(T* p, f32x4 v) {
  typename Vec4<T>::V o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  *reinterpret_cast<typename Vec4<T>::V*>(p) = o;
}
template <int GL>
DEVINL float group_sum(float v) {
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// a lane's place in its head: two runs of 4 values, at o0 and o1
struct Slot {
  int o0, o1;
  bool on, rot;
};
DEVINL Slot slot_of(const FactQkNorm& a, int s) {
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
DEVINL void angles(const NormP& p, int b, int t, int s, f32x4& co, f32x4& si) {
  const int pos = p.a.positions ? p.a.positions[b * p.a.position_stride[0] + t * p.a.position_stride[1]] : p.a.position0 + t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double x = pos * p.turn[min(4 * s + i, 63)];
    x -= rint(x);
    float u, w;
    sincospif((float)(2.0 * x), &u, &w);
    si[i] = u;
    co[i] = w;
  }
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

template <typename T>
DEVINL const T* in_row(const void* q, const int64_t* qs, const void* k, const int64_t* ks, int H, int b, int t, int h) {
  const int64_t* st = h < H ? qs : ks;
  return (const T*)(h < H ? q : k) + b * st[0] + t * st[1] + (h < H ? h : h - H) * st[2];
}

template <typename T, int GL>
__global__ __launch_bounds__(256) void qk_norm_kernel(const NormP p) {
  constexpr int NG = 64 / GL, U = 4;  // heads side by side, and in flight per group
  const FactQkNorm& a = p.a;
  const int lane = threadIdx.x & 63, s = lane % GL, gr = lane / GL, HT = a.H + a.Hkv;
  const long long tok = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tok >= p.tokens) return;
  const int b = (int)(tok / a.n), t = (int)(tok - (long long)b * a.n);
  const Slot sl = slot_of(a, s);
  const bool inter = a.interleaved != 0;
  f32x4 co = {1.f, 1.f, 1.f, 1.f}, si = {0.f, 0.f, 0.f, 0.f};
  f32x4 gq[2], gk[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int o = i ? sl.o1 : sl.o0;
    gq[i] = sl.on && a.q_gamma ? load4(a.q_gamma + o) : f32x4{1.f, 1.f, 1.f, 1.f};
    gk[i] = sl.on && a.k_gamma ? load4(a.k_gamma + o) : f32x4{1.f, 1.f, 1.f, 1.f};
  }
  const float inv = 1.0f / a.dh;
  for (int h0 = 0; h0 < HT; h0 += NG * U) {
    f32x4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * NG + gr;
      x[u] = y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (sl.on && h < HT) {
        const T* r = in_row<T>(a.q, a.q_stride, a.k, a.k_stride, a.H, b, t, h);
        x[u] = load4(r + sl.o0);
        y[u] = load4(r + sl.o1);
      }
    }
    if (h0 == 0 && sl.rot) angles(p, b, t, s, co, si);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * NG + gr;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += x[u][i] * x[u][i] + y[u][i] * y[u][i];
      const float r = rsqrtf(group_sum<GL>(ss) * inv + a.eps);
      if (!sl.on || h >= HT) continue;
      x[u] = x[u] * r * (h < a.H ? gq[0] : gk[0]);
      y[u] = y[u] * r * (h < a.H ? gq[1] : gk[1]);
      if (sl.rot) turn4(x[u], y[u], co, si, inter);
      T* o = const_cast<T*>(in_row<T>(a.q_out, a.q_out_stride, a.k_out, a.k_out_stride, a.H, b, t, h));
      store4(o + sl.o0, x[u]);
      store4(o + sl.o1, y[u]);
    }
  }
}

template <typename T, int GL>
__global__ __launch_bounds__(256) void qk_norm_bwd_kernel(const NormP p) {
  constexpr int NG = 64 / GL, U = 2;
  const FactQkNorm& a = p.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = lane % GL, gr = lane / GL, HT = a.H + a.Hkv;
  const Slot sl = slot_of(a, s);
  const bool inter = a.interleaved != 0;
  f32x4 gq[2], gk[2], aq[2], ak[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int o = i ? sl.o1 : sl.o0;
    gq[i] = sl.on && a.q_gamma ? load4(a.q_gamma + o) : f32x4{1.f, 1.f, 1.f, 1.f};
    gk[i] = sl.on && a.k_gamma ? load4(a.k_gamma + o) : f32x4{1.f, 1.f, 1.f, 1.f};
    aq[i] = ak[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float inv = 1.0f / a.dh;
  for (long long tok = (long long)blockIdx.x * 4 + wave; tok < p.tokens; tok += (long long)gridDim.x * 4) {
    const int b = (int)(tok / a.n), t = (int)(tok - (long long)b * a.n);
    f32x4 co = {1.f, 1.f, 1.f, 1.f}, si = {0.f, 0.f, 0.f, 0.f};
    for (int h0 = 0; h0 < HT; h0 += NG * U) {
      f32x4 x[U][2], d[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * NG + gr;
        x[u][0] = x[u][1] = d[u][0] = d[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (sl.on && h < HT) {
          const T* r = in_row<T>(a.q, a.q_stride, a.k, a.k_stride, a.H, b, t, h);
          x[u][0] = load4(r + sl.o0);
          x[u][1] = load4(r + sl.o1);
          const T* e = in_row<T>(a.dq_out, a.dq_out_stride, a.dk_out, a.dk_out_stride, a.H, b, t, h);
          d[u][0] = load4(e + sl.o0);
          d[u][1] = load4(e + sl.o1);
        }
      }
      if (h0 == 0 && sl.rot) angles(p, b, t, s, co, si);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * NG + gr;
        const bool isq = h < a.H;
        float ss = 0.f, sd = 0.f;
        if (sl.rot) turn4(d[u][0], d[u][1], co, -si, inter);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ss += x[u][i][j] * x[u][i][j];
            sd += x[u][i][j] * d[u][i][j] * (isq ? gq[i][j] : gk[i][j]);
          }
        const float r = rsqrtf(group_sum<GL>(ss) * inv + a.eps);
        const float k = group_sum<GL>(sd) * inv * r * r;
        if (!sl.on || h >= HT) continue;
        T* o = const_cast<T*>(in_row<T>(a.dq, a.dq_stride, a.dk, a.dk_stride, a.H, b, t, h));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4 xr = x[u][i] * r, dg = d[u][i] * xr;
          if (isq) aq[i] += dg;
          else ak[i] += dg;
          store4(o + (i ? sl.o1 : sl.o0), (d[u][i] * (isq ? gq[i] : gk[i]) - x[u][i] * k) * r);
        }
      }
    }
  }
  // gain gradients: the groups of a wave, then the 4 waves, in one order
  __shared__ float red[4][2][128];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = GL; o < 64; o <<= 1) {
        aq[i][j] += __shfl_xor(aq[i][j], o, 64);
        ak[i][j] += __shfl_xor(ak[i][j], o, 64);
      }
  if (gr == 0 && sl.on) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        red[wave][0][(i ? sl.o1 : sl.o0) + j] = aq[i][j];
        red[wave][1][(i ? sl.o1 : sl.o0) + j] = ak[i][j];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dh; i += 256) {
    const int w = i / a.dh, d = i - w * a.dh;
    p.part[(size_t)blockIdx.x * 2 * a.dh + i] = (red[0][w][d] + red[1][w][d]) + (red[2][w][d] + red[3][w][d]);
  }
}

// columns of [rows][2 dh] summed in row order: 16 columns a workgroup, 16 row groups
__global__ __launch_bounds__(256) void qk_norm_dgamma_kernel(const NormP p, int rows) {
  const FactQkNorm& a = p.a;
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, i = blockIdx.x * 16 + c, n = 2 * a.dh;
  __shared__ float red[16][17];
  float x = 0.f;
  if (i < n)
    for (int r = r0; r < rows; r += 16) x += p.part[(size_t)r * n + i];
  red[r0][c] = x;
  __syncthreads();
  if (r0 == 0 && i < n) {
#pragma unroll
    for (int r = 1; r < 16; ++r) x += red[r][c];
    float* o = i < a.dh ? a.dq_gamma : a.dk_gamma;
    if (o) {
      o += i < a.dh ? i : i - a.dh;
      *o = a.dgamma_accumulate ? *o + x : x;
    }
  }
}

int bwd_blocks(const FactQkNorm& a) {
  const long long w = ((long long)a.B * a.n + 3) / 4;
  return (int)(w < 1024 ? w : 1024);
}

NormP params(const FactQkNorm& a) {
  NormP p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.tokens = (long long)a.B * a.n;
  for (int i = 0; i < a.rotary_dim / 2; ++i)
    p.turn[i] = std::pow(a.base, -2.0 * i / a.rotary_dim) / 6.283185307179586476925286766559;
  return p;
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : -100; }

template <typename T, int GL>
int run(const FactQkNorm& a, bool backward, void* ws, hipStream_t s) {
  NormP p = params(a);
  if (!backward) {
    FACT_LAUNCH((qk_norm_kernel<T, GL>), dim3((unsigned)((p.tokens + 3) / 4)), dim3(256), 0, s, p);
    return launched();
  }
  p.part = (float*)ws;
  const int nb = bwd_blocks(a);
  FACT_LAUNCH((qk_norm_bwd_kernel<T, GL>), dim3(nb), dim3(256), 0, s, p);
  if (a.dq_gamma || a.dk_gamma) FACT_LAUNCH(qk_norm_dgamma_kernel, dim3((2 * a.dh + 15) / 16), dim3(256), 0, s, p, nb);
  return launched();
}
template <typename T>
int run(const FactQkNorm& a, bool backward, void* ws, hipStream_t s) {
  if (a.dh <= 32) return run<T, 4>(a, backward, ws, s);
  if (a.dh <= 64) return run<T, 8>(a, backward, ws, s);
  return run<T, 16>(a, backward, ws, s);
}

}  // namespace

int qk_norm_check(const FactQkNorm& a, bool backward, const char** why) {
  auto bad = [&](int rc, const char* w) { *why = w; return rc; };
  if (a.B <= 0 || a.n <= 0 || a.H <= 0 || a.Hkv <= 0) return bad(-1, "B, n, H and Hkv must be positive");
  if ((long long)a.B * a.n > (1ll << 32) || (long long)a.H + a.Hkv > 65536) return bad(-1, "too many tokens or heads");
  if (a.dh < 8 || a.dh > 128 || a.dh % 8) return bad(-3, "unsupported head dim (a multiple of 8 up to 128)");
  if (a.rotary_dim < 0 || a.rotary_dim > a.dh || a.rotary_dim % 8) return bad(-1, "rotary_dim must be a multiple of 8 up to dh");
  if (a.dtype != 0 && a.dtype != 1) return bad(-1, "dtype must be 0 (bf16) or 1 (fp32)");
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
  return 0;
}

size_t qk_norm_ws(const FactQkNorm& a, bool backward) { return backward ? (size_t)bwd_blocks(a) * 2 * a.dh * 4 : 0; }

int launch_qk_norm_fwd(const FactQkNorm& a, hipStream_t s) {
  return a.dtype ? run<float>(a, false, nullptr, s) : run<bf16_t>(a, false, nullptr, s);
}
int launch_qk_norm_bwd(const FactQkNorm& a, void* ws, hipStream_t s) {
  return a.dtype ? run<float>(a, true, ws, s) : run<bf16_t>(a, true, ws, s);
}
