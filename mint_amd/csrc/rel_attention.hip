// Attention with a sliding window, sinks and a learned relative position bias by buckets, forward and backward
// (definition: include/fact_hip.h, FactAttention).
// Times below are of launches under the profiler, each alone between two others; calls one after another take about a tenth less.
//
// Fragment conventions (common.h): scores are computed transposed, S^T = K Q^T, on 16x16x32 bf16 MFMAs, so that one query
// lives in one lane column: lane (g = lane >> 4, c = lane & 15) holds keys 4 g .. 4 g + 3 of query c.  Two stacked 16-key
// score tiles are the B operand of the products that contract over keys (slot j < 4: key 4 g + j, j >= 4: key 16 + 4 g + j - 4),
// their A operands come from the same row-major LDS tiles through the LDS transpose read.  Any [token][head][dh] strides are
// read in place: where dh is no multiple of 32 the last contraction step is padded with zeros in registers and in the LDS rows
// (a 16-deep MFMA costs the same cycles, and one that took up the accumulator right behind a 32-deep one read it too early).
#include "rel_attention.h"

#include <algorithm>
#include <climits>
#include <vector>

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BLOCK_ROWS = 64;  // queries of a workgroup, 16 a wave
constexpr float THR = 6.0f;
constexpr int PAD = 48;  // distances past +-D that a 32 x 16 tile which still touches (-D, D) can reach
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

struct RelP {
  FactAttention a;
  float sc;       // scale * log2 e
  float rscale;   // 1 / scale: the bias enters through the accumulator, which is multiplied by scale afterwards
  int qblocks, nwg;
  int splits;
  int rowtab;     // few rows: the bias of the group's heads fits the workgroup's memory
  int kblocks, sblocks, chunks, schunks;  // dK / dV: blocks of keys, the first of them with sinks, workgroups of a block
  float* dkv;     // partial dK, dV of blocks with several workgroups
  float* dsum;    // [B][H][nq] -rowsum(dO . O)
  float* part;    // per-workgroup bias gradients [H][B][qblocks][2 D + 1] / partial rows of the few-row kernel
};

template <int DH>
struct Geo {
  static constexpr int ND = DH / 16;        // 16-wide head-dim tiles
  static constexpr int KD = (DH + 31) / 32; // 32-deep contraction steps over the head dim
  static constexpr int CH = DH / 8;         // 16-byte chunks of a row
  static constexpr int PC = KD * 4;         // chunks of a row in LDS
  static constexpr int IMG = 32 * PC * 8;   // one 32-row tile (elements)
};
// LDS tiles have no gaps (they are filled 64 chunks at a time); a row's chunks are permuted instead.  A cycle serves 16 chunks of
// 16 bytes, one of each place modulo 16, and rows start PC apart, so rows with the same PC r mod 16 are told apart by `sw`:
//   * a transposed read takes 8 consecutive rows at once, two chunks of each: u differs between them;
//   * a fragment read takes rows 0 .. 3 and 12 .. 15 of one chunk with rows 4 .. 11 of its neighbour: the chunks that either set of
//     rows moves to are whole pairs (u alike, v 0 and 1).
// With u from row & 7 alone the second kind of read took twice the cycles, 30 % of all the LDS was busy.
template <int DH>
struct Swizzle {
  static constexpr int FREE = Geo<DH>::PC == 16 ? 0 : Geo<DH>::PC == 8 ? 1 : 2;  // rows' low bits that PC r tells apart
  static constexpr int MASK = (16 >> FREE) - 1;
};
template <int DH>
DEVINL int place(int row, int ch) {  // element of chunk ch of a row
  constexpr int FREE = Swizzle<DH>::FREE, MASK = Swizzle<DH>::MASK;
  const int v = row >> 3 & 1, u = (row & 7) >> FREE ^ v << (2 - FREE), sw = u << 1 | v;
  return (row * Geo<DH>::PC + (ch & ~MASK) + ((ch & MASK) ^ sw)) * 8;
}
template <int DH>
DEVINL int further(int at, int chunks) {  // place<DH>(row, ch + chunks) from place<DH>(row, ch); no bit is in both ch and chunks
  return (at ^ ((chunks & Swizzle<DH>::MASK) * 8)) + (chunks & ~Swizzle<DH>::MASK) * 8;
}

// one operand fragment set over the head dim: rows of 16 tokens
template <int DH>
struct Frag {
  bf16x8 f[Geo<DH>::KD];
};
template <int DH>
DEVINL void frag_load(Frag<DH>& r, const bf16_t* row, int g) {  // `row`: this lane's row in global memory
#pragma unroll
  for (int kd = 0; kd < Geo<DH>::KD; ++kd) {
    r.f[kd] = zero_bf16x8();
    if (kd * 32 + 32 <= DH || kd * 32 + g * 8 < DH) r.f[kd] = *reinterpret_cast<const bf16x8*>(row + kd * 32 + g * 8);
  }
}
// where a lane's fragments begin in an LDS tile: by rows (row c, chunk g), and through the transpose read
template <int DH>
struct Lane {
  int rows, tr;
  DEVINL void init(int lane) {
    const int g = lane >> 4, s = lane & 15;
    rows = place<DH>(s, g);
    tr = place<DH>(g * 4 + (s >> 2), s >> 1 & 1) + (s & 1) * 4;
  }
};
template <int DH>
DEVINL void frag_lds(Frag<DH>& r, const bf16_t* tile, int sub, int rows) {  // row 16 sub + c
#pragma unroll
  for (int kd = 0; kd < Geo<DH>::KD; ++kd)
    r.f[kd] = *reinterpret_cast<const bf16x8*>(tile + sub * (Geo<DH>::IMG / 2) + further<DH>(rows, kd * 4));
}
template <int DH>
DEVINL f32x4 frag_dot(const Frag<DH>& a, const Frag<DH>& b, f32x4 c) {
#pragma unroll
  for (int kd = 0; kd < Geo<DH>::KD; ++kd) c = mfma16(a.f[kd], b.f[kd], c);
  return c;
}
// zeros into the padding columns of two LDS tiles, once per workgroup
template <int DH>
DEVINL void pad_zero(bf16_t* lds, int tid) {
  using G = Geo<DH>;
  if constexpr (G::PC != G::CH) {
    for (int i = tid; i < 64 * (G::PC - G::CH); i += 256) {
      const int r = i / (G::PC - G::CH);
      *reinterpret_cast<u32x4*>(lds + r / 32 * G::IMG + place<DH>(r % 32, G::CH + i % (G::PC - G::CH))) = u32x4{0u, 0u, 0u, 0u};
    }
  }
}

DEVINL bf16x8 cat4(bf16x4 a, bf16x4 b) { return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
DEVINL bf16x8 pack8(f32x4 a, f32x4 b) {
  return bf16x8{(bf16_t)a[0], (bf16_t)a[1], (bf16_t)a[2], (bf16_t)a[3], (bf16_t)b[0], (bf16_t)b[1], (bf16_t)b[2], (bf16_t)b[3]};
}
// A operand [16 dims of tile dt][32 tokens] of a row-major LDS tile, token slots as in the header comment
template <int DH>
DEVINL bf16x8 frag_tr(const bf16_t* t, int dt, int tr) {
  const bf16_t* p = t + further<DH>(tr, dt * 2);
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)p);
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p + Geo<DH>::IMG / 2));
  return cat4(lo, hi);
}

// x = hi + mid + lo to 24 bits; hi is given
DEVINL void split3(f32x4 a, f32x4 b, const bf16x8& hi, bf16x8& mid, bf16x8& lo) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    a[r] -= (float)hi[r];
    b[r] -= (float)hi[4 + r];
  }
  mid = pack8(a, b);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    a[r] -= (float)mid[r];
    b[r] -= (float)mid[4 + r];
  }
  lo = pack8(a, b);
}

DEVINL float allmax4(float v) {  // over the 4 lanes of a query
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
DEVINL float allsum4(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// ---- which keys a query sees ----------------------------------------------------------------------------------------
struct Vis {
  int len, lo, hi, sinks;  // key j of position p: j < len, j - p <= hi, j - p >= lo or j < sinks
  DEVINL bool seen(int j, int p) const {
    const int d = j - p;  // (selects, no branches: hipcc dropped one of the branchy form's stores)
    return (j < len) & (d <= hi) & ((d >= lo) | (j < sinks));
  }
  DEVINL int count(int p) const {  // of keys that position p sees (saturating sums: hi may be the largest int, lo the smallest)
    const int top = min(len, __builtin_elementwise_add_sat(__builtin_elementwise_add_sat(p, hi), 1));
    const int low = max(0, __builtin_elementwise_add_sat(p, lo)), sk = min(sinks, top);
    return max(0, top - max(low, sk)) + max(0, sk);
  }
  // sees one key only: its softmax is 1 whatever the score, its dS exactly 0 (which P (dP - D) misses by a rounding).  Such a
  // row never lies in a tile that is full.
  DEVINL bool lone(int p) const { return count(p) == 1; }
  // whether one of p .. p + n - 1 may be such a row: over positions the count rises, stays and falls
  DEVINL bool any_lone(int p, int n) const { return count(p) < 2 || count(p + n - 1) < 2; }
  // keys j0 .. j0 + W - 1 against positions p0 .. p0 + R - 1
  template <int W = 32, int R = 32>
  DEVINL bool none(int j0, int p0) const {
    return j0 >= len || j0 - (p0 + R - 1) > hi || (j0 + W - 1 - p0 < lo && j0 >= sinks);
  }
  template <int W = 32, int R = 32>
  DEVINL bool full(int j0, int p0) const {
    return j0 + W - 1 < len && j0 + W - 1 - p0 <= hi && (j0 - (p0 + R - 1) >= lo || j0 + W - 1 < sinks);
  }
};
// Lengths are below 2^30 (checked) and first positions clamped to +-(2^30 - 64), so no key - position overflows.
DEVINL Vis vis_of(const FactAttention& a, int b) {
  Vis v;
  v.len = a.kv_len ? min(max(a.kv_len[b], 0), a.nk) : a.nk;
  v.lo = a.window_left < 0 ? INT_MIN : -a.window_left;
  v.hi = a.window_right < 0 ? INT_MAX : a.window_right;
  v.sinks = a.window_left < 0 ? 0 : a.sinks;
  return v;
}
DEVINL int start_of(const FactAttention& a, int b) {
  return a.q_start ? min(max(a.q_start[b], 64 - (1 << 30)), (1 << 30) - 64) : 0;
}
// the 32-key tiles that positions pa .. pb can see: tiles 0 .. ns - 1 (sinks), then t0 .. t0 + (T - ns) - 1
struct Tiles {
  int ns, t0, T;
  int first, last, sinks;  // keys that any of them sees: first .. last, and up to last those below sinks
  DEVINL int at(int t) const { return t < ns ? t : t - ns + t0; }
  // Rows of a tile that none of them sees are not read, as what is there may be no number, which a probability of zero does not
  // cancel: another row of the tile is taken instead, and masked.
  DEVINL bool whole(int row0) const { return (row0 >= first || row0 + 31 < sinks) && row0 + 31 <= last; }
  DEVINL int row(int row0, int r) const {
    const int j = min(row0 + r, last);
    return (j < first && j >= sinks ? (row0 < sinks ? row0 : first) : j) - row0;
  }
};
DEVINL Tiles tiles_of(const Vis& v, long long pa, long long pb) {
  const long long hi = min((long long)v.len, v.hi == INT_MAX ? (long long)v.len : pb + v.hi + 1);
  const long long lo = v.lo == INT_MIN ? 0 : max(0ll, pa + v.lo);
  Tiles t;
  const int t1 = hi > 0 ? (int)((hi + 31) >> 5) : 0;
  t.ns = hi > 0 ? (int)((min(hi, (long long)v.sinks) + 31) >> 5) : 0;
  t.t0 = max(t.ns, (int)(min(lo, 1ll << 30) >> 5));
  t.T = t.ns + (lo < hi ? max(0, t1 - t.t0) : 0);
  t.first = (int)min(lo, 1ll << 30);
  t.last = (int)hi - 1;
  t.sinks = v.sinks;
  return t;
}

// row of the residual a.out_lo: [B][nq][H][dh] without gaps
DEVINL size_t low_row(const FactAttention& a, int b, int h, int q) { return (((size_t)b * a.nq + q) * a.H + h) * a.dh; }

// Workgroups of one head (and of the heads that share its keys) are neighbours on one XCD (consecutive workgroups go to
// consecutive XCDs): they then read the same K / V rows through one L2.  Speed only.
DEVINL int xcd_order(int id, int n) {
  const int x = id & 7, per = n >> 3, rem = n & 7;
  return (x < rem ? x * (per + 1) : rem * (per + 1) + (x - rem) * per) + (id >> 3);
}

// 16 bytes at a wave-uniform base and a 32-bit byte offset of the lane (one address register; token strides are checked)
DEVINL u32x4 load16(const bf16_t* base, unsigned off) {
  return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) + off);
}

// ---- staging of two 32-row tiles (K and V, or Q and dO) into LDS --------------------------------------------------------
// Loads that write LDS themselves, 16 bytes a lane and 64 consecutive places of a tile an instruction: no registers hold what is
// in flight.  Each wave waits for its own before the barrier (__syncthreads alone does not).  The two buffers of a kernel are two
// objects, each named by half of the unrolled loop: of one array with a computed half the compiler would wait for the loads in
// flight before each read.  At B 8, H 12, n 1440, dh 128 with a bias dK/dV, which took 32 keys a wave then, went from 427 us staged
// through registers to 350 with them; a third buffer, with two tiles in flight, cost the workgroups it left no LDS for (354 instead
// of 263, forward 172 instead of 162, without a bias and in that form as well).
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
template <int DH>
struct Stage {
  using G = Geo<DH>;
  static constexpr int PER = 32 * G::PC / 64, N = PER / 2;  // instructions of a tile; of both tiles and one of the 4 waves
  unsigned off[N];
  unsigned lda, ldb;  // bytes
  int wave, lane;
  DEVINL int tile(int i) const { return i * 4 + wave < PER ? i * 4 + wave : i * 4 + wave - PER; }
  DEVINL int row(int i, int l) const { return (tile(i) * 64 + l) / G::PC; }
  DEVINL int chunk(int i) const {  // (the permutation is its own inverse)
    const int n = tile(i) * 64 + lane, r = n / G::PC;
    return place<DH>(r, n - r * G::PC) / 8 - r * G::PC;
  }
  DEVINL void init(long long a, long long b, int w, int l) {
    lda = (unsigned)a * 2;
    ldb = (unsigned)b * 2;
    wave = w;
    lane = l;
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] = (unsigned)row(i, l) * (i * 4 + wave < PER ? lda : ldb) + chunk(i) * 16;
  }
  // rows row0 .. row0 + 31 of a and b (wave-uniform pointers to row 0)
  DEVINL void load(bf16_t* lds, const bf16_t* a, const bf16_t* b, int row0, const Tiles& t) const {
    a += (long long)row0 * (lda / 2);
    b += (long long)row0 * (ldb / 2);
    if (t.whole(row0)) {
#pragma unroll
      for (int i = 0; i < N; ++i) one(lds, a, b, i, off[i]);
    } else {
      int l = lane;
      asm("" : "+v"(l));  // (rows are worked out here, where they are seldom needed, and hold no registers)
#pragma unroll
      for (int i = 0; i < N; ++i)
        one(lds, a, b, i, off[i] + (unsigned)(t.row(row0, row(i, l)) - row(i, l)) * (i * 4 + wave < PER ? lda : ldb));
    }
  }
  DEVINL void one(bf16_t* lds, const bf16_t* a, const bf16_t* b, int i, unsigned o) const {
    const int k = i * 4 + wave;
    const char* src = reinterpret_cast<const char*>(k < PER ? a : b);
    if (G::PC == G::CH || chunk(i) < G::CH)
      __builtin_amdgcn_global_load_lds((glb_void*)(src + o), (lds_void*)(lds + k * 512), 16, 0, 0);
  }
};

DEVINL void staged() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

// Finite values of the table count up to +-2^14: exp(-2^14) is 0 beside any key that is not hidden as well, and where a row sees
// nothing but such keys its scores keep 2^-10 and less than a step of bf16 of their probabilities.  Further out (1e9 and the type's
// lowest value are what programs hide keys with) value / scale overflows, the rounding of a score is larger than the score, and of
// log-sum-exp = reference point + log2(sum) the second part is lost.  -inf hides a key, NaN stays one.
constexpr float MOST_BIAS = 16384.f;
DEVINL float bias_of(const RelP& p, int i, int h) {  // of head h at place i of the map, divided by scale
  const int bk = min(max(p.a.rel_map[i], 0), p.a.rel_buckets - 1);
  const float x = p.a.rel_table[(size_t)bk * p.a.H + h], y = fabsf(x);
  return ((y > MOST_BIAS) & (y < INFINITY) ? copysignf(MOST_BIAS, x) : x) * p.rscale;
}
// bias of head h for distances -(D + PAD) .. D + PAD, divided by scale
DEVINL void load_bias(float* eb, const RelP& p, int h, int tid, int nthr) {
  const int D = p.a.rel_max_distance;
  for (int i = tid; i < 2 * (D + PAD) + 1; i += nthr) {
    const int d = min(max(i - (D + PAD), -D), D);
    eb[i] = bias_of(p, d + D, h);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// forward: workgroup = 64 queries of one head, 4 waves x 16; 32-key tiles double-buffered in LDS.  One pass over the keys:
//   m' = max(m, s);  l' = l 2^(m - m') + sum 2^(s - m');  O' = O 2^(m - m') + P V;  out = O / l
// In training with a bias vector instructions bound it (60 % of a SIMD's issue, half of them the 24-bit split below; LDS 20 to 27 %,
// matrix pipe below 30 %): B 8, H 12, n 1440, dh 128, all keys 234 us.  Without one no pipe is full (vector 41 to 50 %, LDS 21 to
// 28 %): what bounds it is a tile's dependent chain - scores, exponents, packing, product, one after another in a wave - and the
// barrier every 32 keys: n 8192, H 10, dh 80, window 1023 causal 57 us.  With 32 queries a wave each
// K and V fragment feeds two products, but half as many waves fit, and a block's edge tiles are twice as many: B 4, H 12, n 1440,
// dh 128, window 257 takes 40 us instead of 29, B 8, H 12, n 1440, dh 128, all keys 172 instead of 159.
// ---------------------------------------------------------------------------------------------------------------------
// EXACT (a.out_lo given): the probabilities enter P V as a sum of three bf16 values, 24 bits, and the output's rounding residual
// is kept in fp32.  The backward takes D = rowsum(dO . O) from them: from the rounded P and O it is off by 1e-3 of itself, which
// dS = P (dP - D) and with it the fp32 gradient of the table inherit (two values: 3e-6 of the table's gradient, three: 3e-7).
template <int DH, bool REL, bool EXACT>
__global__ __launch_bounds__(256, 2) void rel_fwd_kernel(const RelP p) {
  using G = Geo<DH>;
  constexpr int ND = G::ND;
  __shared__ __attribute__((aligned(16))) bf16_t buf0[2 * G::IMG], buf1[2 * G::IMG];
  extern __shared__ float eb[];
  const FactAttention& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int id = xcd_order(blockIdx.x, p.nwg);
  const int bh = id / p.qblocks, qb = p.qblocks - 1 - (id - bh * p.qblocks);
  const int b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hkv);
  const Vis v = vis_of(a, b);
  const int start = start_of(a, b);
  const int q0 = qb * BLOCK_ROWS + wave * 16, p0 = start + q0;
  const bool active = q0 < a.nq;
  const Tiles tl = tiles_of(v, (long long)start + qb * BLOCK_ROWS, (long long)start + min(qb * BLOCK_ROWS + BLOCK_ROWS - 1, a.nq - 1));

  Frag<DH> Q;
  frag_load<DH>(Q, (const bf16_t*)a.q + b * a.q_stride[0] + (long long)min(q0 + c, a.nq - 1) * a.q_stride[1] + h * a.q_stride[2], g);
  Lane<DH> at;
  at.init(lane);
  Stage<DH> st;
  const bf16_t* kp = (const bf16_t*)a.k + b * a.k_stride[0] + hk * a.k_stride[2];
  const bf16_t* vp = (const bf16_t*)a.v + b * a.v_stride[0] + hk * a.v_stride[2];
  st.init(a.k_stride[1], a.v_stride[1], wave, lane);
  pad_zero<DH>(buf0, tid);
  pad_zero<DH>(buf1, tid);
  if (tl.T > 0) st.load(buf0, kp, vp, tl.at(0) * 32, tl);
  if (REL) load_bias(eb, p, h, tid, 256);
  f32x4 O[ND];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int D = a.rel_max_distance;
  auto step = [&](int t, const bf16_t* Ks, bf16_t* other) __attribute__((always_inline)) {
    const bf16_t* Vs = Ks + G::IMG;
    const int j0 = tl.at(t) * 32;
    const bool skip = !active || v.none<32, 16>(j0, p0);
    f32x4 s[2];  // key sub-tiles
    if (REL && !skip) {
      const int d0 = j0 - p0;  // distance of the tile's first key and the wave's first query
      if (d0 - 15 >= D || d0 + 31 <= -D) {
        const float f = eb[d0 > 0 ? 2 * (D + PAD) : 0];
        s[0] = s[1] = f32x4{f, f, f, f};
      } else {
        const float* e = eb + d0 + D + PAD + 4 * g - c;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[0][r] = e[r];
          s[1][r] = e[r + 16];
        }
      }
    } else {
      s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (t + 1 < tl.T) st.load(other, kp, vp, tl.at(t + 1) * 32, tl);  // (after the reads of the bias: they would wait for it)
    if (skip) return;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      Frag<DH> K;
      frag_lds<DH>(K, Ks, ks, at.rows);
      s[ks] = frag_dot<DH>(K, Q, s[ks]);
    }
    if (!v.full<32, 16>(j0, p0)) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[ks][r] = v.seen(j0 + ks * 16 + 4 * g + r, p0 + c) ? s[ks][r] : -INFINITY;
    }
    // The reference point m of a row's exponents is raised only when a score passes it by THR powers of two: any m that keeps
    // exp2 in range gives the same softmax, and the common path needs no lane but its own.
    const float mu = m == -INFINITY ? 0.f : m;  // -inf: the row has seen no key yet
    f32x4 x[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[0][r] = fmaf(s[0][r], p.sc, -mu);
      x[1][r] = fmaf(s[1][r], p.sc, -mu);
    }
    const float mx = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                           fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    if (__any((mx > THR) | ((m == -INFINITY) & (mx > -INFINITY)))) {
      const bool first = m == -INFINITY;
      const float top = allmax4(mx);                   // relative to m, or to 0
      const float d = first ? (top == -INFINITY ? 0.f : top) : fmaxf(top, 0.f);
      const float mn = first ? top : m + d;
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l = first ? 0.f : l * alpha;  // (first: nothing has been summed)
      // exponents from the scores again: a reference point far below them, such as that of keys with a bias of -1e9, has left
      // them none of their last bits
      const float mv = mn == -INFINITY ? 0.f : mn;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[0][r] = fmaf(s[0][r], p.sc, -mv);
        x[1][r] = fmaf(s[1][r], p.sc, -mv);
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) O[dt][r] = first ? 0.f : O[dt][r] * alpha;
    }
    f32x4 e0, e1;
    float ls = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      e0[r] = __builtin_amdgcn_exp2f(x[0][r]);
      e1[r] = __builtin_amdgcn_exp2f(x[1][r]);
      ls += e0[r] + e1[r];
    }
    l += ls;
    const bf16x8 pb = pack8(e0, e1);
    bf16x8 pm, pl;
    if (EXACT) split3(e0, e1, pb, pm, pl);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      const bf16x8 vf = frag_tr<DH>(Vs, dt, at.tr);
      O[dt] = mfma16(vf, pb, O[dt]);
      if (EXACT) {
        O[dt] = mfma16(vf, pm, O[dt]);
        O[dt] = mfma16(vf, pl, O[dt]);
      }
    }
  };
  for (int t = 0; t < tl.T;) {
    staged();
    step(t, buf0, buf1);
    if (++t == tl.T) break;
    staged();
    step(t, buf1, buf0);
    ++t;
  }
  const int q = q0 + c;
  const float lt = allsum4(l);
  if (q >= a.nq) return;
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  if (a.lse && g == 0) a.lse[((size_t)b * a.H + h) * a.nq + q] = lt == 0.f ? INFINITY : m + __log2f(lt);
  const long long off = b * a.out_stride[0] + (long long)q * a.out_stride[1] + h * a.out_stride[2] + g * 4;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) {
    bf16x4 o;
    f32x4 lo;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = O[dt][r] * inv;
      o[r] = (bf16_t)x;
      lo[r] = x - (float)o[r];
    }
    *reinterpret_cast<bf16x4*>((bf16_t*)a.out + off + dt * 16) = o;
    if (EXACT) *reinterpret_cast<f32x4*>(a.out_lo + low_row(a, b, h, q) + g * 4 + dt * 16) = lo;
  }
}

// Sums of dS along its diagonals, without atomics.  Of a 16 x 16 sub-tile at base distance d, lane (g, c) holds distances
// d + 4 g + r - c, r = 0 .. 3.
//   * Moving each partial sum one lane on before the next row is added collects a diagonal in one lane: w, lane c, distance
//     d + 4 g + 3 - c.  The three diagonals that leave the 16 lanes come back in lanes 0 .. 2 of the rotated chain: `up`, the same
//     lanes of the sub-tile at d - 16.
//   * The four rows of lanes are 4 distances apart: rows 2 and 3 join rows 0 and 1 moved by 8 lanes, row 1 joins row 0 moved by 4;
//     what leaves on that side belongs to the sub-tile at d + 16.
// Key tiles are visited in ascending order, so a distance is complete after its two neighbours, and row 0 stores 16 of them at a
// time, each once per 16 queries.  At B 8, H 12, n 1440, dh 128 dQ, which took 32 queries a wave when this was chosen, needed 735 us
// with an LDS add per value, 300 with one per folded row (its four rows meet in the same words), 177 without any sums and 214 with
// this.
template <int CTRL, int BANKS = 0xf>
DEVINL float moved(float y) {  // y moved inside rows of 16 lanes; zero from outside and in lanes of other banks of 4
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), CTRL, 0xf, BANKS, true));
}
DEVINL void fold_diagonals(f32x4 v, float& w, float& up) {
  constexpr int SHR1 = 0x111, ROR1 = 0x121;
  w = v[3] + moved<SHR1>(v[2] + moved<SHR1>(v[1] + moved<SHR1>(v[0])));
  up = (v[3] + moved<ROR1>(v[2] + moved<ROR1>(v[1] + moved<ROR1>(v[0])))) - w;
}
struct Diagonals {
  float* bins;         // this wave's sums by distance, 1 - D .. D - 1
  int D, g, c;
  float left, right;   // lane's share of the sums at -D and D
  float w;             // sub-tile at base `at`, without its `up`
  float over1, over2;  // what rows 2, 3 and row 1 of the sub-tile before left for this one
  int at;
  bool open;
  DEVINL float join(float x) {
    constexpr int ROR8 = 0x128, ROR12 = 0x12C;
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto hi = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned h1 = hi[1];
    const float r = __builtin_bit_cast(float, h1);
    const float v = x + moved<ROR8, 0x3>(r) + over1;
    over1 = moved<ROR8, 0xc>(r);
    const unsigned q = __builtin_bit_cast(unsigned, v);
    const auto lo = __builtin_amdgcn_permlane16_swap(q, q, false, false);
    const unsigned l1 = lo[1];
    const float s = __builtin_bit_cast(float, l1);
    const float z = v + moved<ROR12, 0x7>(s) + over2;
    over2 = moved<ROR12, 0x8>(s);
    return z;
  }
  // lane's sum z of distance base + 3 - c (row 0) or further rows', four on each: `fresh` where nothing was stored there before
  DEVINL void put(int base, float z, bool fresh, bool all) {
    const int i = base + (all ? 4 * g : 0) + 3 - c + D - 1;
    if (all || g == 0) {
      if ((i >= 0) & (i < 2 * D - 1)) {
        if (fresh) bins[i] = z;
        else atomicAdd(bins + i, z);
      } else if (i < 0) {
        left += z;
      } else {
        right += z;
      }
    }
  }
  DEVINL void close() {
    if (!open) return;
    put(at, join(w), false, false);  // (where runs of tiles begin and end, a distance can have been stored already)
    put(at + 16, join(0.f), false, false);
    open = false;
  }
  // the sub-tiles at bases d0, d0 + 16
  DEVINL void tile(int d0, f32x4 a, f32x4 b) {
    float wa, ua, wb, ub;
    const bool on = open && at + 16 == d0;
    if (!on) close();
    fold_diagonals(a, wa, ua);
    fold_diagonals(b, wb, ub);
    if (on) {
      put(d0 - 16, join(w + ua), true, false);
      put(d0, join(wa + ub), true, false);
    } else {  // (`ua` reaches into the 16 distances stored before it)
      over1 = over2 = 0.f;
      put(d0, join(wa + ub), true, false);
      put(d0 - 16, ua, false, true);
    }
    w = wb;
    at = d0 + 16;
    open = true;
  }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward dQ and the bias gradient: workgroup = 64 queries of one head, 16 a wave
//   P = exp2(S c - L);  dP = V dO^T;  dS = P (dP - D), D = rowsum(dO . O);  dQ^T += K^T dS;  dbias[j - p] += dS
// Bound by the tile's dependent chain and its barrier: no pipe is above 45 % (vector 45 % at dh 80 with a bias, 39 at dh 64, 27 at
// dh 128 without one and 2.4 waves a SIMD; LDS 17 to 33 %, matrix pipe 25 %).  B 8, H 12, n 1440, dh 128, all keys with a bias: 266 us,
// B 4, window 257 without one: 41.  32 queries a wave: 49 us
// instead of 38 (B 4, H 12, n 1440, dh 128, window 257), 231 instead of 237 where nothing but full tiles is left (B 8, all keys).
// ---------------------------------------------------------------------------------------------------------------------
template <int DH, bool REL>
__global__ __launch_bounds__(256, DH > 96 ? 3 : 4) void rel_dq_kernel(const RelP p) {
  using G = Geo<DH>;
  constexpr int ND = G::ND;
  __shared__ __attribute__((aligned(16))) bf16_t buf0[2 * G::IMG], buf1[2 * G::IMG];
  extern __shared__ float eb[];
  const FactAttention& a = p.a;
  const int D = a.rel_max_distance, NB = 2 * (D + PAD) + 1;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float* bins = eb + NB + (2 * D - 1) * wave;  // this wave's bias gradient by distance: its own, so sums have one order
  const int id = xcd_order(blockIdx.x, p.nwg);
  const int bh = id / p.qblocks, qb = p.qblocks - 1 - (id - bh * p.qblocks);
  const int b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hkv);
  const Vis v = vis_of(a, b);
  const int start = start_of(a, b);
  const int q0 = qb * BLOCK_ROWS + wave * 16, p0 = start + q0;
  const bool active = q0 < a.nq;
  const Tiles tl = tiles_of(v, (long long)start + qb * BLOCK_ROWS, (long long)start + min(qb * BLOCK_ROWS + BLOCK_ROWS - 1, a.nq - 1));

  Lane<DH> at;
  at.init(lane);
  Stage<DH> st;
  const bf16_t* kp = (const bf16_t*)a.k + b * a.k_stride[0] + hk * a.k_stride[2];
  const bf16_t* vp = (const bf16_t*)a.v + b * a.v_stride[0] + hk * a.v_stride[2];
  st.init(a.k_stride[1], a.v_stride[1], wave, lane);
  pad_zero<DH>(buf0, tid);
  pad_zero<DH>(buf1, tid);
  if (tl.T > 0) st.load(buf0, kp, vp, tl.at(0) * 32, tl);
  const int q = min(q0 + c, a.nq - 1);
  const bool live = (q0 + c < a.nq) & !v.lone(start + q);  // a query of the call that sees more than one key
  Frag<DH> Q, dO;
  frag_load<DH>(Q, (const bf16_t*)a.q + b * a.q_stride[0] + (long long)q * a.q_stride[1] + h * a.q_stride[2], g);
  frag_load<DH>(dO, (const bf16_t*)a.dout + b * a.dout_stride[0] + (long long)q * a.dout_stride[1] + h * a.dout_stride[2], g);
  float part = 0.f;
  {
    Frag<DH> f;
    frag_load<DH>(f, (const bf16_t*)a.out + b * a.out_stride[0] + (long long)q * a.out_stride[1] + h * a.out_stride[2], g);
#pragma unroll
    for (int kd = 0; kd < G::KD; ++kd)
#pragma unroll
      for (int j = 0; j < 8; ++j) part += (float)dO.f[kd][j] * (float)f.f[kd][j];
    if (a.out_lo) {
      const float* lo = a.out_lo + low_row(a, b, h, q);
#pragma unroll
      for (int kd = 0; kd < G::KD; ++kd)
        if (kd * 32 + 32 <= DH || kd * 32 + g * 8 < DH) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(lo + kd * 32 + g * 8);
          const f32x4 y = *reinterpret_cast<const f32x4*>(lo + kd * 32 + g * 8 + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) part += (float)dO.f[kd][j] * x[j] + (float)dO.f[kd][4 + j] * y[j];
        }
    }
  }
  part = allsum4(part);
  const size_t row = ((size_t)b * a.H + h) * a.nq + q;
  const float nL = -a.lse[row];
  if (active && g == 0) p.dsum[row] = -part;  // for the dK / dV kernel (repeated rows write the same value)
  // Every second wave carries its queries with the sign turned over (dS, hence dQ): the matrix pipe adds with a rounding that
  // leans down by 0.02 of a last place, which the millions of dS behind one table entry add up to 3.5e-6 of its gradient.
  const bool turned = wave & 1;
  const float nD = turned ? part : -part;
  if (turned) {
#pragma unroll
    for (int kd = 0; kd < G::KD; ++kd) dO.f[kd] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, dO.f[kd]) ^ 0x80008000u);
  }
  f32x4 dQ[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) dQ[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  Diagonals diag;
  diag.bins = bins;
  diag.D = D;
  diag.g = g;
  diag.c = c;
  diag.left = diag.right = 0.f;
  diag.over1 = diag.over2 = 0.f;
  diag.open = false;
  diag.w = 0.f;
  diag.at = 0;
  if (REL) {
    load_bias(eb, p, h, tid, 256);
    for (int i = lane; i < 2 * D - 1; i += 64) bins[i] = 0.f;
  }
  auto step = [&](int t, const bf16_t* Ks, bf16_t* other) __attribute__((always_inline)) {
    const bf16_t* Vs = Ks + G::IMG;
    const int j0 = tl.at(t) * 32;
    const bool skip = !active || v.none<32, 16>(j0, p0);
    f32x4 s[2], dp[2];
    const int d0 = j0 - p0;
    const bool left = REL && d0 + 31 <= -D, right = REL && d0 - 15 >= D;
    if (REL && !skip) {
      if (left || right) {
        const float f = eb[right ? NB - 1 : 0];
        s[0] = s[1] = f32x4{f, f, f, f};
      } else {
        const float* e = eb + d0 + D + PAD + 4 * g - c;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[0][r] = e[r];
          s[1][r] = e[r + 16];
        }
      }
    } else {
      s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (t + 1 < tl.T) st.load(other, kp, vp, tl.at(t + 1) * 32, tl);  // (after the reads of the bias: they would wait for it)
    if (skip) return;
    f32x4 ds[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      Frag<DH> K, V;
      frag_lds<DH>(K, Ks, ks, at.rows);
      frag_lds<DH>(V, Vs, ks, at.rows);
      dp[ks] = f32x4{nD, nD, nD, nD};
      s[ks] = frag_dot<DH>(K, Q, s[ks]);
      dp[ks] = frag_dot<DH>(V, dO, dp[ks]);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int r = 0; r < 4; ++r) ds[ks][r] = __builtin_amdgcn_exp2f(fmaf(s[ks][r], p.sc, nL)) * dp[ks][r];
    if (!v.full<32, 16>(j0, p0) || q0 + 15 >= a.nq) {  // (queries past the last repeat it: kept out of the bias gradient)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int r = 0; r < 4; ++r) ds[ks][r] = (v.seen(j0 + ks * 16 + 4 * g + r, p0 + c) & live) ? ds[ks][r] : 0.f;
    }
    const bf16x8 dsb = pack8(ds[0], ds[1]);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) dQ[dt] = mfma16(frag_tr<DH>(Ks, dt, at.tr), dsb, dQ[dt]);
    if (REL) {
      if (left || right) {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) x += ds[0][r] + ds[1][r];
        if (left) diag.left += x;
        else diag.right += x;
      } else {
        diag.tile(d0, ds[0], ds[1]);
      }
    }
  };
  for (int t = 0; t < tl.T;) {
    staged();
    step(t, buf0, buf1);
    if (++t == tl.T) break;
    staged();
    step(t, buf1, buf0);
    ++t;
  }
  if (q0 + c < a.nq) {
    bf16_t* out = (bf16_t*)a.dq + b * a.dq_stride[0] + (long long)q * a.dq_stride[1] + h * a.dq_stride[2] + g * 4;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      bf16x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (bf16_t)(dQ[dt][r] * (turned ? -a.scale : a.scale));
      *reinterpret_cast<bf16x4*>(out + dt * 16) = o;
    }
  }
  if (REL) {
    diag.close();
    const float far[2] = {wave_sum(diag.left), wave_sum(diag.right)};
    __syncthreads();
    if (lane == 0) eb[wave] = far[0], eb[4 + wave] = far[1];  // (the table is not read any more)
    __syncthreads();
    float* out = p.part + (((size_t)h * a.B + b) * p.qblocks + qb) * (2 * D + 1);
    const float* b0 = eb + NB;
    const int n = 2 * D - 1;
    for (int i = tid; i < n; i += 256) out[1 + i] = (b0[i] + b0[2 * n + i]) - (b0[n + i] + b0[3 * n + i]);
    if (tid < 2) out[tid * 2 * D] = (eb[4 * tid] + eb[4 * tid + 2]) - (eb[4 * tid + 1] + eb[4 * tid + 3]);
  }
}

// drel[bucket][h], a workgroup each: the distances of the bucket, listed in order, over the batch and the query blocks.  B 8, H 12,
// n 1440, 64 buckets of 1025 distances: 9 MB in 15 us, as long as its largest bucket takes.
__global__ __launch_bounds__(256) void rel_dtable_kernel(const RelP p) {
  const FactAttention& a = p.a;
  const int D = a.rel_max_distance, n = 2 * D + 1, h = blockIdx.x, bu = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ short list[2049 + 63];
  __shared__ int counts[4];
  __shared__ float red[4];
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + tid;
    const bool in = i < n && min(max(a.rel_map[min(i, n - 1)], 0), a.rel_buckets - 1) == bu;
    const unsigned long long m = __ballot(in);
    if (lane == 0) counts[wave] = __popcll(m);
    __syncthreads();
    int at = total;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += counts[w];
      total += counts[w];
    }
    if (in) list[at + __popcll(m & ((1ull << lane) - 1))] = (short)i;
    __syncthreads();
  }
  // 8 groups of 32 threads, every 8th row each: four rows' loads are under way at once
  const int rows = a.B * p.qblocks, first = tid >> 5;
  const float* part = p.part + (size_t)h * rows * n;
  float x = 0.f;
  for (int i = tid & 31; i < total; i += 32) {
    const float* col = part + list[i];
    int r = first;
    for (; r + 24 < rows; r += 32) {
      const float y0 = col[(size_t)r * n], y1 = col[(size_t)(r + 8) * n], y2 = col[(size_t)(r + 16) * n], y3 = col[(size_t)(r + 24) * n];
      x += (y0 + y1) + (y2 + y3);
    }
    for (; r < rows; r += 8) x += col[(size_t)r * n];
  }
  x = wave_sum(x);
  if (lane == 0) red[wave] = x;
  __syncthreads();
  if (tid == 0) {
    x = (red[0] + red[1]) + (red[2] + red[3]);
    float* o = a.drel + (size_t)bu * a.H + h;
    *o = a.drel_accumulate ? *o + x : x;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// backward dK / dV: workgroup = 64 keys of one key head, 4 waves x 16; the query tiles of every head that reads them are
// streamed (heads of a group one after another).  A block's stream is cut into `chunks` workgroups where there are too few
// blocks to fill the chip or a block holds sinks, which all later queries see: their fp32 sums go through the workspace and
// rel_join_dkdv_kernel adds them in order.
// ---------------------------------------------------------------------------------------------------------------------
struct KBlock {
  int bh, kb, chunk, chunks;
  int slot;  // index among the chunks that go through the workspace, -1: the block is written directly
};
// grid: per (b, key head) first the blocks with sinks (p.schunks workgroups each), then the others (p.chunks each)
DEVINL KBlock kblock_of(const RelP& p, int id) {
  const int per = p.sblocks * p.schunks + (p.kblocks - p.sblocks) * p.chunks;
  const int through = (p.schunks > 1 ? p.sblocks * p.schunks : 0) + (p.chunks > 1 ? (p.kblocks - p.sblocks) * p.chunks : 0);
  KBlock k;
  k.bh = id / per;
  int r = id - k.bh * per;
  if (r < p.sblocks * p.schunks) {
    k.kb = r / p.schunks;
    k.chunks = p.schunks;
    k.chunk = r - k.kb * p.schunks;
    k.slot = p.schunks > 1 ? k.bh * through + r : -1;
  } else {
    r -= p.sblocks * p.schunks;
    k.kb = p.sblocks + r / p.chunks;
    k.chunks = p.chunks;
    k.chunk = r % p.chunks;
    k.slot = p.chunks > 1 ? k.bh * through + (p.schunks > 1 ? p.sblocks * p.schunks : 0) + r : -1;
  }
  return k;
}

// A wave has 16 keys and its four sums fit the registers of 4 (dh 128: 3) workgroups a CU.  With 32 keys a wave every Q and dO
// fragment feeds two products, but two workgroups a CU are left: dh 64, B 2, H 12 on 4 key heads, n 2047, window 256 took 45.8 us
// against 29.8; B 4, H 12, n 1440, window 257: 57 against 38; B 8, H 12, n 1440, all keys: 186 against 176 (dh 80: 222 and 214,
// dh 32: 115 and 132, the one that lost).  What is left is latency, as in dQ: vector issue 26 to 40 %, LDS 21 to 40 %, matrix pipe
// 18 %.  B 8, H 12, n 1440, dh 128, all keys with a bias: 305 us; B 4, window 257 without one: 56 and the join 5.
constexpr int BLOCK_KEYS = 64;
constexpr int dkdv_slots(int dh) { return dh <= 96 ? 4 : 3; }  // workgroups of a CU
template <int DH, bool REL>
__global__ __launch_bounds__(256, dkdv_slots(DH)) void rel_dkdv_kernel(const RelP p) {
  using G = Geo<DH>;
  constexpr int ND = G::ND;
  __shared__ __attribute__((aligned(16))) bf16_t buf0[2 * G::IMG + 128], buf1[2 * G::IMG + 128];  // Q, dO, fp32 L and -D
  extern __shared__ float eb[];
  const FactAttention& a = p.a;
  const int D = a.rel_max_distance, NB = 2 * (D + PAD) + 1;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.H / a.Hkv;
  const KBlock blk = kblock_of(p, xcd_order(blockIdx.x, p.nwg));
  const int kb = blk.kb, b = blk.bh / a.Hkv, hk = blk.bh - b * a.Hkv;
  const Vis v = vis_of(a, b);
  const int start = start_of(a, b);
  const int j0 = kb * BLOCK_KEYS + wave * 16;
  const bool active = j0 < v.len;
  // query rows that see any key of the block: positions [ka - hi, ke - lo], or all later ones if it holds a sink
  const long long ka = kb * BLOCK_KEYS, ke = min(kb * BLOCK_KEYS + BLOCK_KEYS - 1, v.len - 1);
  long long qa = v.hi == INT_MAX ? 0 : max(0ll, ka - v.hi - start);
  long long qe = (v.lo == INT_MIN || ka < v.sinks) ? a.nq - 1 : min((long long)a.nq - 1, ke - v.lo - start);
  if (ka >= v.len) qe = -1;
  const int t0 = (int)(min(qa, 1ll << 30) >> 5), T = qe >= qa ? (int)(qe >> 5) - t0 + 1 : 0, TT = T * group;
  const int per = (TT + blk.chunks - 1) / blk.chunks, ib = min(TT, blk.chunk * per), ie = min(TT, ib + per);

  Frag<DH> K, V;
  {
    const long long j = max(0, min(j0 + c, v.len - 1));
    frag_load<DH>(K, (const bf16_t*)a.k + b * a.k_stride[0] + j * a.k_stride[1] + hk * a.k_stride[2], g);
    frag_load<DH>(V, (const bf16_t*)a.v + b * a.v_stride[0] + j * a.v_stride[1] + hk * a.v_stride[2], g);
  }
  pad_zero<DH>(buf0, tid);
  pad_zero<DH>(buf1, tid);
  f32x4 dK[ND], dV[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) dK[dt] = dV[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  Lane<DH> at;
  at.init(lane);
  Stage<DH> st;
  st.init(a.q_stride[1], a.dout_stride[1], wave, lane);
  const Tiles all = {0, 0, 0, 0, a.nq - 1, 0};
  auto load = [&](int hh, int qt, bf16_t* buf) __attribute__((always_inline)) {  // head hh of the group, its query tile t0 + qt
    const int h = hk * group + hh, q0 = (t0 + qt) * 32;
    st.load(buf, (const bf16_t*)a.q + b * a.q_stride[0] + h * a.q_stride[2],
            (const bf16_t*)a.dout + b * a.dout_stride[0] + h * a.dout_stride[2], q0, all);
    if (wave == 0) {
      int l = lane;
      asm("" : "+v"(l));  // (the addresses are made here, not kept)
      const size_t row = ((size_t)b * a.H + h) * a.nq + min(q0 + (l & 31), a.nq - 1);
      __builtin_amdgcn_global_load_lds((glb_void*)((l < 32 ? a.lse : p.dsum) + row), (lds_void*)(buf + 2 * G::IMG), 4, 0, 0);
    }
  };
  int hh = ib < ie ? ib / T : 0, qt = ib - hh * T;
  if (ib < ie) load(hh, qt, buf0);
  auto step = [&](int i, const bf16_t* Qs, bf16_t* other) __attribute__((always_inline)) {
    if (REL && (qt == 0 || i == ib)) {  // the next head's bias: after the last tile of the head before has been read
      __syncthreads();
      load_bias(eb, p, hk * group + hh, tid, 256);
    }
    staged();
    const bf16_t* Os = Qs + G::IMG;
    const float* sl = reinterpret_cast<const float*>(Qs + 2 * G::IMG);
    const int q0 = (t0 + qt) * 32, p0 = start + q0;
    const bool skip = !active || v.none<16>(j0, p0);
    if (DH >= 80) asm("" : "+v"(at.tr));  // offsets made from them each tile: kept, they do not fit the registers
    if (DH >= 80 && (REL || DH < 96)) asm("" : "+v"(at.rows));
    f32x4 s[2], dp[2];  // query sub-tiles: lane = key c, queries 4 g .. 4 g + 3
    if (REL && !skip) {
      const int d0 = j0 - p0;
      if (d0 - 31 >= D || d0 + 15 <= -D) {
        const float f = eb[d0 > 0 ? NB - 1 : 0];
        s[0] = s[1] = f32x4{f, f, f, f};
      } else {
        const float* e = eb + d0 + D + PAD + c - 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[0][r] = e[-r];
          s[1][r] = e[-r - 16];
        }
      }
    } else {
      s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (++qt == T) {
      qt = 0;
      ++hh;
    }
    if (i + 1 < ie) load(hh, qt, other);  // (after the reads of the bias: they would wait for it)
    if (skip) return;
    f32x4 L[2], pr[2];
#pragma unroll
    for (int qs = 0; qs < 2; ++qs) {
      L[qs] = *reinterpret_cast<const f32x4*>(sl + qs * 16 + g * 4);
      dp[qs] = *reinterpret_cast<const f32x4*>(sl + 32 + qs * 16 + g * 4);
      Frag<DH> Q, dO;
      frag_lds<DH>(Q, Qs, qs, at.rows);
      frag_lds<DH>(dO, Os, qs, at.rows);
      s[qs] = frag_dot<DH>(Q, K, s[qs]);
      dp[qs] = frag_dot<DH>(dO, V, dp[qs]);
    }
#pragma unroll
    for (int qs = 0; qs < 2; ++qs)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        pr[qs][r] = __builtin_amdgcn_exp2f(fmaf(s[qs][r], p.sc, -L[qs][r]));
        dp[qs][r] *= pr[qs][r];
      }
    if (!v.full<16>(j0, p0) || q0 + 31 >= a.nq) {
#pragma unroll
      for (int qs = 0; qs < 2; ++qs)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int q = qs * 16 + 4 * g + r;
          const bool ok = v.seen(j0 + c, p0 + q) & (q0 + q < a.nq);
          pr[qs][r] = ok ? pr[qs][r] : 0.f;
          dp[qs][r] = ok ? dp[qs][r] : 0.f;
        }
      if (v.any_lone(p0, 32)) {
#pragma unroll
        for (int qs = 0; qs < 2; ++qs)
#pragma unroll
          for (int r = 0; r < 4; ++r) dp[qs][r] = v.lone(p0 + qs * 16 + 4 * g + r) ? 0.f : dp[qs][r];
      }
    }
    const bf16x8 pb = pack8(pr[0], pr[1]), db = pack8(dp[0], dp[1]);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      dV[dt] = mfma16(frag_tr<DH>(Os, dt, at.tr), pb, dV[dt]);
      dK[dt] = mfma16(frag_tr<DH>(Qs, dt, at.tr), db, dK[dt]);
    }
  };
  for (int i = ib; i < ie;) {
    step(i, buf0, buf1);
    if (++i == ie) break;
    step(i, buf1, buf0);
    ++i;
  }
  if (blk.slot >= 0) {
    f32x4* out = reinterpret_cast<f32x4*>(p.dkv) + ((size_t)blk.slot * (BLOCK_KEYS / 16) + wave) * (2 * ND * 64) + lane;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      out[dt * 128] = dK[dt];
      out[dt * 128 + 64] = dV[dt];
    }
    return;
  }
  const int j = j0 + c;
  if (j >= a.nk) return;
  bf16_t* kr = (bf16_t*)a.dk + b * a.dk_stride[0] + (long long)j * a.dk_stride[1] + hk * a.dk_stride[2] + g * 4;
  bf16_t* vr = (bf16_t*)a.dv + b * a.dv_stride[0] + (long long)j * a.dv_stride[1] + hk * a.dv_stride[2] + g * 4;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) {
    bf16x4 x, y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = (bf16_t)(dK[dt][r] * a.scale);
      y[r] = (bf16_t)dV[dt][r];
    }
    *reinterpret_cast<bf16x4*>(kr + dt * 16) = x;
    *reinterpret_cast<bf16x4*>(vr + dt * 16) = y;
  }
}

// the chunks of a block, in order: a wave per accumulator fragment (16-key sub-tile, dt, K or V) of the kernel above
template <int DH>
__global__ __launch_bounds__(256) void rel_join_dkdv_kernel(const RelP p) {
  constexpr int ND = Geo<DH>::ND, FR = BLOCK_KEYS / 16 * 2 * ND;  // fragments of a block
  const FactAttention& a = p.a;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int f = (blockIdx.x * 4 + (threadIdx.x >> 6)) % FR, blk = (blockIdx.x * 4 + (threadIdx.x >> 6)) / FR;
  const int sj = p.schunks > 1 ? p.sblocks : 0, oj = p.chunks > 1 ? p.kblocks - p.sblocks : 0;
  if (blk >= a.B * a.Hkv * (sj + oj)) return;
  const int bh = blk / (sj + oj), r = blk - bh * (sj + oj), b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const bool sink = r < sj;
  const int kb = sink ? r : p.sblocks + r - sj, n = sink ? p.schunks : p.chunks;
  const int slot = bh * (sj * p.schunks + oj * p.chunks) + (sink ? r * p.schunks : sj * p.schunks + (r - sj) * p.chunks);
  const f32x4* src = reinterpret_cast<const f32x4*>(p.dkv) + ((size_t)slot * FR + f) * 64 + lane;
  f32x4 x = src[0];
  for (int i = 1; i < n; ++i) x += src[(size_t)i * FR * 64];
  const int dt = (f >> 1) % ND, isv = f & 1;
  const int j = kb * BLOCK_KEYS + f / (2 * ND) * 16 + c;
  if (j >= a.nk) return;
  const int64_t* st = isv ? a.dv_stride : a.dk_stride;
  const float k = isv ? 1.f : a.scale;
  bf16x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (bf16_t)(x[i] * k);
  *reinterpret_cast<bf16x4*>((bf16_t*)(isv ? a.dv : a.dk) + b * st[0] + (long long)j * st[1] + hk * st[2] + dt * 16 + g * 4) = o;
}

// ---------------------------------------------------------------------------------------------------------------------
// few rows: all nq * group <= 16 query rows of one key head are the 16 columns of a score tile; the waves of a workgroup and
// the splits of a head take different key tiles and are joined by their maxima and sums at the end.  Bound by the reads of K and V:
// 4 sequences of 16384 .. 32767 keys, H 10, dh 80 (315 MB) take 72 us, 4.4 TB/s; a small call (B 32, H 10, 360 keys, 37 MB) 12.4 us,
// of which a third is the chain of length, tile, score, probability, output and join.
// ---------------------------------------------------------------------------------------------------------------------
template <int DH, bool REL>
__global__ __launch_bounds__(256, 2) void rel_rows_kernel(const RelP p) {
  using G = Geo<DH>;
  constexpr int ND = G::ND, NV = G::CH / 2;  // 16-byte chunks of V a lane moves per 32-key tile
  constexpr int DEPTH = DH > 96 ? 1 : 2;     // tiles in flight a wave: two of dh 128 do not fit 256 registers
  constexpr int OP = DH + 4;                 // pitch of the joined rows (floats)
  constexpr int BYTES = 4 * 16 * OP * 4 > 4 * G::IMG * 2 ? 4 * 16 * OP * 4 : 4 * G::IMG * 2;
  __shared__ __attribute__((aligned(16))) unsigned char smem[BYTES];
  __shared__ float ml[4][2][16];
  extern __shared__ float tab[];  // bias of the group's heads by distance, if p.rowtab
  const FactAttention& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // key heads of one range of tokens beside each other on one XCD: their rows share cache lines
  const int id = p.splits > 1 ? (int)blockIdx.x : xcd_order(blockIdx.x, p.nwg);
  const int bs = id / a.Hkv, hk = id - bs * a.Hkv, b = bs / p.splits, split = bs - b * p.splits;
  const int group = a.H / a.Hkv, R = group * a.nq;
  const Vis v = vis_of(a, b);
  const int start = start_of(a, b);
  const Tiles tl = tiles_of(v, start, (long long)start + a.nq - 1);
  const int row = min(c, R - 1), h = hk * group + row / a.nq, qi = row - (row / a.nq) * a.nq, pos = start + qi;
  Frag<DH> Q;
  frag_load<DH>(Q, (const bf16_t*)a.q + b * a.q_stride[0] + (long long)qi * a.q_stride[1] + h * a.q_stride[2], g);
  const int per = (tl.T + p.splits - 1) / p.splits;
  const int tb = split * per, te = min(tl.T, tb + per);
  const bf16_t* kb = (const bf16_t*)a.k + b * a.k_stride[0] + hk * a.k_stride[2];
  const bf16_t* vb = (const bf16_t*)a.v + b * a.v_stride[0] + hk * a.v_stride[2];
  bf16_t* Vs = reinterpret_cast<bf16_t*>(smem) + wave * G::IMG;
  Lane<DH> at;
  at.init(lane);
  const int D = a.rel_max_distance, n = 2 * D + 1, hr = row / a.nq;
  auto bias = [&](int head, int i) { return bias_of(p, i, head); };  // distance i - D

  struct Tile {  // one 32-key tile in flight: K as fragments, V as rows
    Frag<DH> K[2];
    u32x4 vr[NV];
  } tile[DEPTH];
  const unsigned ldk = (unsigned)a.k_stride[1] * 2, ldv = (unsigned)a.v_stride[1] * 2;
  auto load = [&](Tile& x, int t) {
    const int j0 = tl.at(t) * 32;
    const bool whole = tl.whole(j0);
    const bf16_t* k0 = kb + (long long)j0 * a.k_stride[1];
    const bf16_t* v0 = vb + (long long)j0 * a.v_stride[1];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const unsigned r = whole ? ks * 16 + c : tl.row(j0, ks * 16 + c);
#pragma unroll
      for (int kd = 0; kd < G::KD; ++kd) {
        x.K[ks].f[kd] = zero_bf16x8();
        if (kd * 32 + 32 <= DH || kd * 32 + g * 8 < DH)
          x.K[ks].f[kd] = __builtin_bit_cast(bf16x8, load16(k0, r * ldk + kd * 64 + g * 16));
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = lane + i * 64, r = q / G::CH, ch = q - r * G::CH;
      x.vr[i] = load16(v0, (unsigned)(whole ? r : tl.row(j0, r)) * ldv + ch * 16);
    }
  };
  f32x4 O[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DEPTH; ++i)
    if (tb + wave + 4 * i < te) load(tile[i], tb + wave + 4 * i);
  float left = 0.f, right = 0.f;
  if (REL) {
    left = bias(h, 0);
    right = bias(h, n - 1);
    // the table, where this workgroup's tiles come nearer than D to a row
    if (p.rowtab && tb < te && tl.at(tb) * 32 - (start + a.nq - 1) < D && tl.at(te - 1) * 32 + 31 - start > -D) {
      for (int i = tid; i < group * n; i += 256) tab[i] = bias(hk * group + i / n, i % n);
      __syncthreads();
    }
  }
  auto step = [&](Tile& x, int t) {
    const int j0 = tl.at(t) * 32;
    f32x4 s[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) s[ks] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (REL) {
      if (j0 + 31 - start <= -D || j0 - (start + a.nq - 1) >= D) {
        const float f = j0 < start ? left : right;
        s[0] = s[1] = f32x4{f, f, f, f};
      } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = min(max(j0 + ks * 16 + 4 * g + r - pos, -D), D) + D;
            s[ks][r] = p.rowtab ? tab[hr * n + i] : bias(h, i);
          }
      }
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) s[ks] = frag_dot<DH>(x.K[ks], Q, s[ks]);
    // (all rows lie in the 16 positions from start on)
    if (!(j0 + 31 < v.len && j0 + 31 - start <= v.hi && (j0 - (start + a.nq - 1) >= v.lo || j0 + 31 < v.sinks))) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[ks][r] = v.seen(j0 + ks * 16 + 4 * g + r, pos) ? s[ks][r] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = lane + i * 64, r = q / G::CH, ch = q - r * G::CH;
      *reinterpret_cast<u32x4*>(Vs + place<DH>(r, ch)) = x.vr[i];
    }
    if (t + 4 * DEPTH < te) load(x, t + 4 * DEPTH);
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = allmax4(mx) * p.sc;
    const float mn = fmaxf(m, mx);
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    const float mu = mn == -INFINITY ? 0.f : mn;
    m = mn;
    f32x4 e0, e1;
    float ls = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      e0[r] = __builtin_amdgcn_exp2f(fmaf(s[0][r], p.sc, -mu));
      e1[r] = __builtin_amdgcn_exp2f(fmaf(s[1][r], p.sc, -mu));
      ls += e0[r] + e1[r];
    }
    l = l * alpha + ls;
    const bf16x8 pb = pack8(e0, e1);
    bf16x8 pm = zero_bf16x8(), pl = zero_bf16x8();
    if (a.out_lo) split3(e0, e1, pb, pm, pl);  // as in the forward above
    __builtin_amdgcn_wave_barrier();  // the tile below was written by this wave alone: its LDS accesses stay in order
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
      const bf16x8 vf = frag_tr<DH>(Vs, dt, at.tr);
      O[dt] = mfma16(vf, pb, O[dt] * alpha);
      if (a.out_lo) {
        O[dt] = mfma16(vf, pm, O[dt]);
        O[dt] = mfma16(vf, pl, O[dt]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  for (int t = tb + wave; t < te; t += 4 * DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (t + 4 * i < te) step(tile[i], t + 4 * i);
  }
  l = allsum4(l);
  __syncthreads();
  float* Oj = reinterpret_cast<float*>(smem);
  if (g == 0) {
    ml[wave][0][c] = m;
    ml[wave][1][c] = l;
  }
#pragma unroll
  for (int dt = 0; dt < ND; ++dt) *reinterpret_cast<f32x4*>(Oj + (wave * 16 + c) * OP + dt * 16 + g * 4) = O[dt];
  __syncthreads();
  // join the 4 waves: a thread takes 4 dims of a row
  for (int i = tid; i < R * (DH / 4); i += 256) {
    const int r = i / (DH / 4), d = (i - r * (DH / 4)) * 4;
    float M = fmaxf(fmaxf(ml[0][0][r], ml[1][0][r]), fmaxf(ml[2][0][r], ml[3][0][r]));
    const float mu = M == -INFINITY ? 0.f : M;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[w][0][r] - mu);
      lt += ml[w][1][r] * f;
      o += *reinterpret_cast<const f32x4*>(Oj + (w * 16 + r) * OP + d) * f;
    }
    if (p.splits > 1) {
      float* out = p.part + (((size_t)(b * a.Hkv + hk) * p.splits + split) * R + r) * (DH + 4);
      if (d == 0) {
        out[0] = M;
        out[1] = lt;
      }
      *reinterpret_cast<f32x4*>(out + 4 + d) = o;
    } else {
      const int hh = hk * group + r / a.nq, q = r - (r / a.nq) * a.nq;
      const float inv = lt == 0.f ? 0.f : 1.0f / lt;
      if (a.lse && d == 0) a.lse[((size_t)b * a.H + hh) * a.nq + q] = lt == 0.f ? INFINITY : M + __log2f(lt);
      const long long off = b * a.out_stride[0] + (long long)q * a.out_stride[1] + hh * a.out_stride[2] + d;
      bf16x4 x;
      f32x4 y;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = (bf16_t)(o[k] * inv);
        y[k] = o[k] * inv - (float)x[k];
      }
      *reinterpret_cast<bf16x4*>((bf16_t*)a.out + off) = x;
      if (a.out_lo) *reinterpret_cast<f32x4*>(a.out_lo + low_row(a, b, hh, q) + d) = y;
    }
  }
}

// join the splits of the few-row kernel: a workgroup per row, every 4th split a wave, 2 dims a lane
__global__ __launch_bounds__(256) void rel_join_kernel(const RelP p) {
  const FactAttention& a = p.a;
  const int group = a.H / a.Hkv, R = group * a.nq, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bh = blockIdx.x / R, r = blockIdx.x - bh * R, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const size_t pitch = a.dh + 4, step = (size_t)R * pitch;
  const float* src = p.part + ((size_t)bh * p.splits * R + r) * pitch;
  __shared__ float red[2][4], f[256];
  __shared__ f32x2 o[4][64];
  const float m = tid < p.splits ? src[tid * step] : -INFINITY, l = tid < p.splits ? src[tid * step + 1] : 0.f;  // splits <= 256
  const int d = min(lane * 2, a.dh - 2);
  float M = wave_max(m);
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  f[tid] = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
  const float lw = wave_sum(l * f[tid]);
  if (lane == 0) red[1][wave] = lw;
  __syncthreads();
  f32x2 x = {0.f, 0.f};
#pragma unroll 4
  for (int s = wave; s < p.splits; s += 4) {
    const f32x2 y = *reinterpret_cast<const f32x2*>(src + s * step + 4 + d);
    x[0] = fmaf(y[0], f[s], x[0]);
    x[1] = fmaf(y[1], f[s], x[1]);
  }
  o[wave][lane] = x;
  __syncthreads();
  if (wave) return;
  const float lt = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int h = hk * group + r / a.nq, q = r - (r / a.nq) * a.nq;
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  if (a.lse && lane == 0) a.lse[((size_t)b * a.H + h) * a.nq + q] = lt == 0.f ? INFINITY : M + __log2f(lt);
  if (lane * 2 >= a.dh) return;
  const float o0 = ((o[0][lane][0] + o[1][lane][0]) + (o[2][lane][0] + o[3][lane][0])) * inv;
  const float o1 = ((o[0][lane][1] + o[1][lane][1]) + (o[2][lane][1] + o[3][lane][1])) * inv;
  const bf16x2 y = {(bf16_t)o0, (bf16_t)o1};
  *reinterpret_cast<bf16x2*>((bf16_t*)a.out + b * a.out_stride[0] + (long long)q * a.out_stride[1] + h * a.out_stride[2] + d) = y;
  if (a.out_lo) *reinterpret_cast<f32x2*>(a.out_lo + low_row(a, b, h, q) + d) = f32x2{o0 - (float)y[0], o1 - (float)y[1]};
}

__global__ __launch_bounds__(256) void zero_rows_kernel(bf16_t* x, int n, int t0, int ld, int chunks, long long total) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / chunks;
    const long long b = r / (n - t0), t = t0 + r - b * (n - t0);
    *reinterpret_cast<u32x4*>(x + (b * n + t) * ld + (i - r * chunks) * 8) = u32x4{0u, 0u, 0u, 0u};
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
int launched() { return hipGetLastError() == hipSuccess ? 0 : -100; }

// more than 64 KiB of LDS has to be allowed once per kernel and device
template <typename K>
int allow_lds(K kernel, size_t dynamic, size_t fixed) {
  if (dynamic + fixed <= 65536) return 0;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             (int)dynamic) == hipSuccess ? 0 : -101;
}

bool few_rows(const FactAttention& a) { return (long long)a.nq * (a.H / a.Hkv) <= 16; }

// keys that one sequence's rows can see at most
long long span(const FactAttention& a) {
  if (a.window_left < 0) return a.nk;
  const long long right = a.window_right < 0 ? a.nk : a.window_right;
  return std::min<long long>(a.nk, (long long)a.window_left + right + a.nq + a.sinks + 62);
}

// splits of the few-row kernel: up to 1536 workgroups - of sequences of 16384 to 32767 keys at B 4, H 10, dh 80 the rows take 72 us,
// with 512 (as many as run at once) 77, the longest sequence's being the last - of at least 8 tiles (2 a wave) each: with half as
// many tiles a workgroup, B 32 and 4 key heads over 1028 keys of dh 128 take 20 us instead of 17.5
int row_splits(const FactAttention& a) {
  const long long tiles = (span(a) + 31) / 32, wgs = (long long)a.B * a.Hkv;
  long long s = std::min((1536 + wgs - 1) / wgs, tiles / 8);
  return (int)std::max(1ll, std::min(s, 256ll));
}

size_t up16(size_t x) { return (x + 15) & ~(size_t)15; }

constexpr long long SLOTS = 768;  // workgroups that run at once at dh 128 (more do at smaller ones; cut for 1024, they take longer)

RelP params(const FactAttention& a) {
  RelP p;
  p.a = a;
  p.sc = a.scale * LOG2E;
  p.rscale = 1.0f / a.scale;
  p.qblocks = (a.nq + BLOCK_ROWS - 1) / BLOCK_ROWS;
  p.nwg = 0;
  p.splits = 1;
  p.rowtab = 0;
  p.dsum = nullptr;
  p.part = nullptr;
  p.dkv = nullptr;
  // dK / dV: streams of the blocks as long as lengths and positions allow (they are on the device), cut so that the chip
  // is filled but no piece is shorter than 4 tiles
  const long long group = a.H / a.Hkv, all = ((long long)a.nq + 31) / 32 * group;
  p.kblocks = (a.nk + BLOCK_KEYS - 1) / BLOCK_KEYS;
  p.sblocks = a.window_left < 0 ? 0 : (std::min(a.sinks, a.nk) + BLOCK_KEYS - 1) / BLOCK_KEYS;
  long long seen = a.nq;
  if (a.window_left >= 0 && a.window_right >= 0)
    seen = std::min<long long>(seen, (long long)BLOCK_KEYS + a.window_left + a.window_right + 62);
  const long long t = (seen + 31) / 32 * group, blocks = (long long)a.B * a.Hkv * p.kblocks;
  p.chunks = (int)std::max(1ll, std::min((SLOTS + blocks / 2) / blocks, t / 4));
  // blocks with sinks, which all later queries see: pieces as long as the other blocks', or, where there is much other work to
  // run beside them, a quarter of a workgroup slot's share of the whole
  const long long share = ((long long)(p.kblocks - p.sblocks) * t + p.sblocks * all) * a.B * a.Hkv / (4 * SLOTS);
  const long long piece = std::max({8ll, (t + p.chunks - 1) / p.chunks, share});
  p.schunks = (int)std::max<long long>(p.chunks, std::min(all / piece, 64ll));
  return p;
}
// chunks of one (batch, key head) that go through the workspace
size_t dkv_chunks(const RelP& p) {
  return (p.schunks > 1 ? (size_t)p.sblocks * p.schunks : 0) + (p.chunks > 1 ? (size_t)(p.kblocks - p.sblocks) * p.chunks : 0);
}
size_t dkv_bytes(const RelP& p) { return dkv_chunks(p) * p.a.B * p.a.Hkv * BLOCK_KEYS * 2 * p.a.dh * 4; }

// the dQ kernel's partial bias gradients
size_t part_bytes(const FactAttention& a) {
  return a.rel_table ? up16((size_t)a.B * a.H * ((a.nq + BLOCK_ROWS - 1) / BLOCK_ROWS) * (2 * a.rel_max_distance + 1) * 4) : 0;
}

template <int DH, bool REL>
int fwd_t(const FactAttention& a, void* ws, hipStream_t s) {
  RelP p = params(a);
  if (few_rows(a)) {
    p.splits = row_splits(a);
    p.part = (float*)ws;
    p.nwg = p.splits * a.B * a.Hkv;
    const size_t tab = (size_t)(a.H / a.Hkv) * (2 * a.rel_max_distance + 1) * 4;
    p.rowtab = REL && tab <= 16384;
    FACT_LAUNCH((rel_rows_kernel<DH, REL>), dim3(p.nwg), dim3(256), p.rowtab ? tab : 0, s, p);
    if (p.splits > 1) FACT_LAUNCH(rel_join_kernel, dim3(a.B * a.H * a.nq), dim3(256), 0, s, p);
    return launched();
  }
  p.nwg = p.qblocks * a.B * a.H;
  const size_t lds = REL ? (2 * (a.rel_max_distance + PAD) + 1) * 4 : 0;
  auto go = [&](auto kernel) {
    FACT_LAUNCH(kernel, dim3(p.nwg), dim3(256), lds, s, p);
    return launched();
  };
  return a.out_lo ? go(rel_fwd_kernel<DH, REL, true>) : go(rel_fwd_kernel<DH, REL, false>);
}

template <int DH, bool REL>
int bwd_t(const FactAttention& a, void* ws, hipStream_t s) {
  RelP p = params(a);
  const size_t nb = REL ? 2 * (a.rel_max_distance + PAD) + 1 : 0;
  p.dsum = (float*)ws;
  p.part = (float*)((char*)ws + up16((size_t)a.B * a.H * a.nq * 4));
  p.dkv = (float*)((char*)p.part + part_bytes(a));
  p.nwg = p.qblocks * a.B * a.H;
  const size_t lds1 = (nb + (REL ? 4 * (2 * a.rel_max_distance - 1) : 0)) * 4, lds2 = nb * 4;
  if (int rc = allow_lds(rel_dq_kernel<DH, REL>, lds1, 4 * Geo<DH>::IMG * 2)) return rc;
  FACT_LAUNCH((rel_dq_kernel<DH, REL>), dim3(p.nwg), dim3(256), lds1, s, p);
  if (REL) FACT_LAUNCH(rel_dtable_kernel, dim3(a.H, a.rel_buckets), dim3(256), 0, s, p);
  p.nwg = (p.sblocks * p.schunks + (p.kblocks - p.sblocks) * p.chunks) * a.B * a.Hkv;
  FACT_LAUNCH((rel_dkdv_kernel<DH, REL>), dim3(p.nwg), dim3(256), lds2, s, p);
  const int joined = ((p.schunks > 1 ? p.sblocks : 0) + (p.chunks > 1 ? p.kblocks - p.sblocks : 0)) * a.B * a.Hkv;
  if (joined) FACT_LAUNCH(rel_join_dkdv_kernel<DH>, dim3(joined * (BLOCK_KEYS / 32) * Geo<DH>::ND), dim3(256), 0, s, p);
  return launched();
}

template <int DH>
int run(const FactAttention& a, bool backward, void* ws, hipStream_t s) {
  if (backward) return a.rel_table ? bwd_t<DH, true>(a, ws, s) : bwd_t<DH, false>(a, ws, s);
  return a.rel_table ? fwd_t<DH, true>(a, ws, s) : fwd_t<DH, false>(a, ws, s);
}
int run(const FactAttention& a, bool backward, void* ws, hipStream_t s) {
  switch (a.dh) {
    case 32: return run<32>(a, backward, ws, s);
    case 64: return run<64>(a, backward, ws, s);
    case 80: return run<80>(a, backward, ws, s);
    case 96: return run<96>(a, backward, ws, s);
    case 128: return run<128>(a, backward, ws, s);
  }
  return -10;
}

}  // namespace

int rel_attention_check(const FactAttention& a, bool backward, const char** why) {
  auto bad = [&](int rc, const char* w) { *why = w; return rc; };
  const int big = 1 << 30;
  if (a.B <= 0 || a.H <= 0 || a.Hkv <= 0 || a.nq <= 0 || a.nk <= 0) return bad(-1, "B, H, Hkv, nq and nk must be positive");
  if (a.nq >= big || a.nk >= big) return bad(-1, "nq and nk must be below 2^30");
  if (a.H % a.Hkv) return bad(-1, "H must be a multiple of Hkv");
  if (a.dh != 32 && a.dh != 64 && a.dh != 80 && a.dh != 96 && a.dh != 128)
    return bad(-3, "unsupported head dim (supported: 32, 64, 80, 96, 128)");
  // (a launch has fewer than 2^32 threads, 256 a workgroup)
  const long long most = (1 << 24) - 1, heads = (long long)a.B * a.H;
  if (heads > most || (a.nq + 63ll) / 64 * heads > most || (few_rows(a) && a.nq * heads > most) ||
      (backward && (a.nk + 63ll) / 64 * a.B * a.Hkv > most / 64))
    return bad(-1, "too many heads and blocks for one launch");
  if (!(a.scale >= 5.9604645e-8f) || !(a.scale <= 3.0e38f)) return bad(-1, "scale must be finite and at least 2^-24");
  if (a.sinks < 0) return bad(-1, "sinks must not be negative");
  if (a.rel_table) {
    if (!a.rel_map) return bad(-1, "rel_table needs rel_map");
    if (a.rel_buckets < 1 || a.rel_buckets > 256) return bad(-1, "rel_buckets must be 1..256");
    if (a.rel_max_distance < 1 || a.rel_max_distance > 1024) return bad(-1, "rel_max_distance must be 1..1024");
  }
  struct T { const void* p; const int64_t* st; bool out; };
  const T t[] = {{a.q, a.q_stride, false}, {a.k, a.k_stride, false}, {a.v, a.v_stride, false}, {a.out, a.out_stride, !backward},
                 {a.dout, a.dout_stride, false}, {a.dq, a.dq_stride, true}, {a.dk, a.dk_stride, true}, {a.dv, a.dv_stride, true}};
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    if (!t[i].p) return bad(-1, "null tensor");
    if ((uintptr_t)t[i].p & 15) return bad(-1, "tensors must be 16-byte aligned");
    // (tiles of 32 rows are addressed with 32-bit byte offsets)
    if (t[i].st[1] < 0 || t[i].st[1] > 1 << 25) return bad(-1, "token strides must be 0..2^25 elements");
    for (int k = 0; k < 3; ++k) {
      if (t[i].st[k] & 7) return bad(-1, "strides must be multiples of 8 elements");
      const int n[3] = {a.B, i == 1 || i == 2 || i == 6 || i == 7 ? a.nk : a.nq, i == 1 || i == 2 || i == 6 || i == 7 ? a.Hkv : a.H};
      if (t[i].out && t[i].st[k] == 0 && n[k] > 1) return bad(-1, "an output must not be broadcast");
    }
  }
  // (`out` may be q: a workgroup reads its own rows before it writes them, if they are the same)
  for (int i = 0; i < (backward ? 8 : 4); ++i)
    for (int k = 0; k < i; ++k) {
      if (t[i].p != t[k].p || !(t[i].out || t[k].out)) continue;
      const int n[3] = {a.B, a.nq, a.H};
      bool place = i == 3 && k == 0;
      for (int j = 0; j < 3; ++j) place = place && (n[j] == 1 || t[i].st[j] == t[k].st[j]);
      if (!place) return bad(-1, "an output must not be another tensor (but `out` may be q, with the same strides)");
    }
  const void* more[] = {a.out_lo, a.lse, a.drel, a.rel_table, a.rel_map, a.kv_len, a.q_start};
  for (int i = 0; i < 7; ++i) {
    if (!more[i]) continue;
    const bool out = backward ? i == 2 : i < 2;
    for (int k = 0; k < (backward ? 8 : 4); ++k)
      if (more[i] == t[k].p && (out || t[k].out)) return bad(-1, "an output must not be another tensor");
    for (int k = 0; k < 7; ++k)
      if (out && k != i && more[i] == more[k]) return bad(-1, "an output must not be another tensor");
  }
  if ((uintptr_t)a.out_lo & 15) return bad(-1, "tensors must be 16-byte aligned");
  if (backward && !a.lse) return bad(-1, "the backward needs the forward's lse");
  if (backward && a.rel_table && !a.drel) return bad(-1, "the backward with rel_table needs drel");
  return 0;
}

size_t rel_attention_ws(const FactAttention& a, bool backward) {
  if (backward) return up16((size_t)a.B * a.H * a.nq * 4) + part_bytes(a) + dkv_bytes(params(a));
  if (!few_rows(a)) return 0;
  const int s = row_splits(a);
  return s > 1 ? up16((size_t)s * a.B * a.H * a.nq * (a.dh + 4) * 4) : 0;
}

int launch_zero_rows(bf16_t* x, int B, int n, int t0, int ld, int width, hipStream_t s) {
  if (width & 7 || ld & 7 || (uintptr_t)x & 15) return -1;
  const long long total = (long long)B * (n - t0) * (width / 8);
  if (total <= 0) return 0;
  FACT_LAUNCH(zero_rows_kernel, dim3((unsigned)std::min<long long>((total + 255) / 256, 4096)), dim3(256), 0, s, x, n, t0, ld,
              width / 8, total);
  return launched();
}

int launch_rel_attention_fwd(const FactAttention& a, void* ws, hipStream_t s) { return run(a, false, ws, s); }
int launch_rel_attention_bwd(const FactAttention& a, void* ws, hipStream_t s) { return run(a, true, ws, s); }

namespace {
// little-endian base-2^32 number times a small one
void times(std::vector<uint32_t>& x, uint32_t m) {
  uint64_t carry = 0;
  for (uint32_t& w : x) {
    carry += (uint64_t)w * m;
    w = (uint32_t)carry;
    carry >>= 32;
  }
  if (carry) x.push_back((uint32_t)carry);
}
bool not_less(const std::vector<uint32_t>& x, const std::vector<uint32_t>& y) {
  if (x.size() != y.size()) return x.size() > y.size();
  for (size_t i = x.size(); i-- > 0;)
    if (x[i] != y[i]) return x[i] > y[i];
  return true;
}
}  // namespace

// floor(log(d / e) / log(D / e) * w) >= t  <=>  d^w e^t >= D^t e^w, with e = exact buckets and w the logarithmic ones
int relative_buckets(int num_buckets, int max_distance, int bidirectional, int32_t* map) {
  const int n = bidirectional ? num_buckets / 2 : num_buckets, e = n / 2, w = n - e;
  if (!map || num_buckets > 256 || n < 2 || (bidirectional && (num_buckets & 1)) || max_distance <= e || max_distance > 1024)
    return -1;
  std::vector<int> side(max_distance + 1);
  for (int d = 0; d <= max_distance; ++d) {
    if (d < e) {
      side[d] = d;
      continue;
    }
    int t = d > e ? side[d - 1] - e : 0;  // (buckets do not fall with the distance)
    while (t + 1 < w) {
      std::vector<uint32_t> x(1, 1), y(1, 1);
      for (int i = 0; i < w; ++i) { times(x, d); times(y, e); }
      for (int i = 0; i < t + 1; ++i) { times(x, e); times(y, max_distance); }
      if (!not_less(x, y)) break;
      ++t;
    }
    side[d] = e + t;
  }
  for (int d = -max_distance; d <= max_distance; ++d) {
    int b = d > 0 ? (bidirectional ? n + side[d] : 0) : side[-d];
    map[d + max_distance] = b;
  }
  return 0;
}
