// Per-head RMS norm of queries and keys and the position rotation, in one pass over the rows, forward and backward.
//   forward : y = R(pos) (x r w),  r = rsqrt(mean(x^2) + eps)
//   backward: g = R(pos)^T dy,  h = g w,  dx = r (h - x r mean(h x r)),  dw = sum over tokens and heads of g x r
// r is recomputed from x, which the backward reads anyway.  Bound by memory: a row is read and written once, in 16-byte
// pieces; sums are fp32.  A row (one head of one token) belongs to L neighbouring lanes, and a lane holds the two 8-element
// chunks that the rotation pairs up (i and i + R/2, or two neighbouring chunks), so that turning a pair never crosses lanes
// and only the sum of squares does.  A wave keeps the angles of its token(s) in registers while it walks over their heads.
// Forward, 131072 tokens of 16 heads of 64, queries and keys in bf16 (1.07 GB): 212 us, 5.1 TB/s, the rate of a large copy;
// 20001 tokens of 8 heads of 128, 32 elements rotated, positions in no order: 29 us.
#include "common.hpp"

namespace pdt {

constexpr int QR_WAVES = 4;

struct QrLane {  // what a lane owns of every row
  int c0, c1;    // its two chunks (16-byte pieces)
  bool ok0, ok1, turn0, turn1;
  int a0, a1;    // first angle of each chunk
};
// MODE 0: no rotation, 1: pairs (i, i + R/2), 2: neighbouring pairs
template <int MODE>
__device__ __forceinline__ QrLane qr_lane(const PdtQkRope& p, int slot) {
  const int chunks = p.D >> 3, pairs = MODE == 1 ? p.R >> 4 : 0;
  QrLane l;
  if (slot < pairs) {
    l.c0 = slot; l.c1 = slot + pairs;
    l.a0 = l.a1 = slot * 8;
  } else {
    l.c0 = 2 * slot; l.c1 = 2 * slot + 1;  // (behind the pairs: 2 pairs + 2 (slot - pairs))
    l.a0 = l.c0 * 4; l.a1 = l.c1 * 4;
  }
  l.ok0 = l.c0 < chunks; l.ok1 = l.c1 < chunks;
  l.turn0 = MODE == 1 ? slot < pairs : (MODE == 2 && l.c0 * 8 < p.R);
  l.turn1 = MODE == 1 ? slot < pairs : (MODE == 2 && l.c1 * 8 < p.R);
  return l;
}
template <typename T>
__device__ __forceinline__ void qr_fetch(const T* row, const QrLane& l, short8& va, short8& vb) {
  const short8 none = {0, 0, 0, 0, 0, 0, 0, 0};
  va = vb = none;
  if (l.ok0) va = *reinterpret_cast<const short8*>(row + l.c0 * 8);
  if (l.ok1) vb = *reinterpret_cast<const short8*>(row + l.c1 * 8);
}
template <typename T>
__device__ __forceinline__ void qr_load(const T* row, const QrLane& l, float (&a)[8], float (&b)[8]) {
  short8 va, vb;
  qr_fetch<T>(row, l, va, vb);
  unpack8<T>(va, a);
  unpack8<T>(vb, b);
}
template <typename T>
__device__ __forceinline__ void qr_store(T* row, const QrLane& l, const float (&a)[8], const float (&b)[8]) {
  if (l.ok0) *reinterpret_cast<short8*>(row + l.c0 * 8) = pack8<T>(a);
  if (l.ok1) *reinterpret_cast<short8*>(row + l.c1 * 8) = pack8<T>(b);
}
// angles of the lane's pairs: MODE 1 eight (cs[e] turns (a[e], b[e])), MODE 2 four per chunk (cs[i] turns (a[2i], a[2i+1]),
// cs[4 + i] turns (b[2i], b[2i+1])); chunks that are not turned get angle 0
template <int MODE>
__device__ __forceinline__ void qr_angles(const PdtQkRope& p, const QrLane& l, int64_t pos, float (&cs)[8], float (&sn)[8]) {
  const int64_t at = pos * (p.R >> 1);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool turn = h ? l.turn1 : l.turn0;
    const int64_t i = at + (MODE == 1 ? l.a0 + 4 * h : (h ? l.a1 : l.a0));
    float4v c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
    if (turn) {
      c = *reinterpret_cast<const float4v*>(p.cos + i);
      s = *reinterpret_cast<const float4v*>(p.sin + i);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { cs[4 * h + e] = c[e]; sn[4 * h + e] = s[e]; }
  }
}
// turns the lane's pairs by the angles (DIR 1) or back (DIR -1)
template <int MODE, int DIR>
__device__ __forceinline__ void qr_turn(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8]) {
  if (MODE == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = a[e], y = b[e], s = DIR * sn[e];
      a[e] = x * cs[e] - y * s;
      b[e] = y * cs[e] + x * s;
    }
  } else if (MODE == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = a[2 * i], y = a[2 * i + 1], s = DIR * sn[i];
      a[2 * i] = x * cs[i] - y * s;
      a[2 * i + 1] = y * cs[i] + x * s;
      const float z = b[2 * i], w = b[2 * i + 1], t = DIR * sn[4 + i];
      b[2 * i] = z * cs[4 + i] - w * t;
      b[2 * i + 1] = w * cs[4 + i] + z * t;
    }
  }
}
template <int L>
__device__ __forceinline__ float qr_sum(float v) {  // over the L lanes of a row
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <typename T>
__device__ __forceinline__ void qr_weight(const PdtQkRope& p, int side, const QrLane& l, float (&wa)[8], float (&wb)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) wa[e] = wb[e] = 0.f;
  if (!p.w[side]) return;
  if (p.w_f32) {
    const float* w = (const float*)p.w[side];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (l.ok0) wa[e] = w[l.c0 * 8 + e];
      if (l.ok1) wb[e] = w[l.c1 * 8 + e];
    }
  } else {
    qr_load<T>((const T*)p.w[side], l, wa, wb);
  }
}
__device__ __forceinline__ int64_t qr_pos(const PdtQkRope& p, int t, int at) {
  const int64_t i = p.pos ? p.pos[t] : at;
  return i < 0 ? 0 : (i >= p.P ? p.P - 1 : i);
}
template <typename T>
__device__ __forceinline__ T* qr_row(const PdtRelView& v, int b, int at) { return (T*)v.p + (int64_t)b * v.batch + (int64_t)at * v.row; }

// Groups of L lanes: GT of them (a power of two, at most the heads of the wider side) share a token
template <typename T, int L, int MODE>
__global__ __launch_bounds__(64 * QR_WAVES) void qk_rope_fwd_kernel(PdtQkRope p, int gt) {
  const int lane = threadIdx.x & 63, grp = lane / L;
  const int per_wave = (64 / L) / gt;  // tokens of a wave
  const QrLane l = qr_lane<MODE>(p, lane & (L - 1));
  const int t = (blockIdx.x * QR_WAVES + (threadIdx.x >> 6)) * per_wave + grp / gt;
  if (t >= p.T) return;
  const int b = t / p.seq, at = t - b * p.seq;
  float cs[8], sn[8];
  if (MODE) qr_angles<MODE>(p, l, qr_pos(p, t, at), cs, sn);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const T* x = qr_row<const T>(p.x[side], b, at);
    T* y = qr_row<T>(p.y[side], b, at);
    float wa[8], wb[8];
    qr_weight<T>(p, side, l, wa, wb);
    for (int h = grp & (gt - 1); h < p.heads[side]; h += gt) {
      float a[8], c[8];
      qr_load<T>(x + (int64_t)h * p.x[side].head, l, a, c);
      if (p.w[side]) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + c[e] * c[e];
        const float r = rsqrtf(qr_sum<L>(ss) / p.D + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) { a[e] *= r * wa[e]; c[e] *= r * wb[e]; }
      }
      qr_turn<MODE, 1>(a, c, cs, sn);
      qr_store<T>(y + (int64_t)h * p.y[side].head, l, a, c);
    }
  }
}

// Grid-stride over the tokens, so that the weight gradient stays in registers: a lane adds up its 16 columns, the workgroup
// writes one partial row.  blockIdx.y = side: with both sides in one workgroup the two weights and two sums cost 64 registers
// more.  The 144 to 166 registers (forced under 128 they spill: 530 us) leave 3 waves per SIMD, so loads run one item ahead,
// and the grid is what fits the card at once, 768 workgroups over both sides.  131072 tokens of 16 heads of 64 (1.61 GB):
// 326 us, 4.9 TB/s.  Loading one item at a time took 390 us, 1024 workgroups (one round and a third) 378 us.
constexpr int QR_BWD_BLOCKS = 384;
template <typename T, int L, int MODE>
__global__ __launch_bounds__(64 * QR_WAVES) void qk_rope_bwd_kernel(PdtQkRope p, int gt, float* __restrict__ partial) {
  __shared__ float red[QR_WAVES][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane / L, side = blockIdx.y;
  const int per_wave = (64 / L) / gt;
  const QrLane l = qr_lane<MODE>(p, lane & (L - 1));
  const bool normed = p.w[side] != nullptr;
  float acc_a[8], acc_b[8], wa[8], wb[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc_a[e] = acc_b[e] = 0.f;
  qr_weight<T>(p, side, l, wa, wb);
  // one (token, head) after the other; the next one's rows and position are on their way while this one is worked on
  const int step = gridDim.x * QR_WAVES * per_wave, heads = p.heads[side], h0 = grp & (gt - 1);
  int t = h0 < heads ? (blockIdx.x * QR_WAVES + wave) * per_wave + grp / gt : p.T, h = h0, turned = -1;
  short8 x0, x1, g0, g1;
  int64_t pos = 0;
  const auto fetch = [&](int tn, int hn) {
    const int b = tn / p.seq, at = tn - b * p.seq;
    if (normed) qr_fetch<T>(qr_row<const T>(p.x[side], b, at) + (int64_t)hn * p.x[side].head, l, x0, x1);
    qr_fetch<T>(qr_row<const T>(p.y[side], b, at) + (int64_t)hn * p.y[side].head, l, g0, g1);
    if (MODE) pos = qr_pos(p, tn, at);
  };
  if (t < p.T) fetch(t, h);
  float cs[8], sn[8];
  while (t < p.T) {
    float xa[8], xb[8], ga[8], gb[8];
    unpack8<T>(g0, ga);
    unpack8<T>(g1, gb);
    if (normed) {
      unpack8<T>(x0, xa);
      unpack8<T>(x1, xb);
    }
    if (MODE && turned != t) qr_angles<MODE>(p, l, pos, cs, sn);
    turned = t;
    const int b = t / p.seq, at = t - b * p.seq;
    T* dx = qr_row<T>(p.dx[side], b, at) + (int64_t)h * p.dx[side].head;
    h += gt;
    if (h >= heads) { h = h0; t += step; }
    if (t < p.T) fetch(t, h);
    qr_turn<MODE, -1>(ga, gb, cs, sn);
    if (normed) {
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss += xa[e] * xa[e] + xb[e] * xb[e];
        dot += ga[e] * wa[e] * xa[e] + gb[e] * wb[e] * xb[e];
      }
      const float r = rsqrtf(qr_sum<L>(ss) / p.D + p.eps);
      const float m = qr_sum<L>(dot) * r * r / p.D;  // mean(h x r) r
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc_a[e] += ga[e] * xa[e] * r;
        acc_b[e] += gb[e] * xb[e] * r;
        ga[e] = r * (ga[e] * wa[e] - xa[e] * m);
        gb[e] = r * (gb[e] * wb[e] - xb[e] * m);
      }
    }
    qr_store<T>(dx, l, ga, gb);
  }
  if (!partial) return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int o = 32; o >= L; o >>= 1) {
      acc_a[e] += __shfl_xor(acc_a[e], o, 64);
      acc_b[e] += __shfl_xor(acc_b[e], o, 64);
    }
  if (lane < L) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (l.ok0) red[wave][l.c0 * 8 + e] = acc_a[e];
      if (l.ok1) red[wave][l.c1 * 8 + e] = acc_b[e];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += 64 * QR_WAVES) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < QR_WAVES; ++v) s += red[v][c];
    partial[((int64_t)blockIdx.x * 2 + side) * p.D + c] = s;
  }
}

static int qr_lanes(const PdtQkRope& p) {  // lanes per row: a power of two that holds all chunk pairs
  const int pairs = p.interleaved ? 0 : p.R >> 4;
  const int slots = pairs + (((p.D >> 3) - 2 * pairs) + 1) / 2;
  int l = 1;
  while (l < slots) l *= 2;
  return l;
}
static int qr_groups(const PdtQkRope& p, int lanes) {
  const int heads = p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1];
  int g = 1;
  while (g < heads && g < 64 / lanes) g *= 2;
  return g;
}
static int qr_check(int dtype, const PdtQkRope& p, bool bwd) {
  if (dtype != PDT_F16 && dtype != PDT_BF16) return -1;
  if (p.T < 0 || p.T > (1 << 30) || p.seq <= 0 || p.heads[0] < 0 || p.heads[1] < 0 || p.D <= 0 || p.D > 256 || p.D % 8) return -3;
  if (p.R < 0 || p.R > p.D || p.R % (p.interleaved ? 8 : 16)) return -3;
  if (p.R && (!p.cos || !p.sin || p.P <= 0 || (uintptr_t)p.cos % 16 || (uintptr_t)p.sin % 16)) return -2;
  for (int i = 0; i < 2; ++i) {
    const PdtRelView* v[3] = {&p.x[i], &p.y[i], &p.dx[i]};
    for (int j = 0; j < (bwd ? 3 : 2); ++j)
      if (p.heads[i] && p.T &&
          (!v[j]->p || (uintptr_t)v[j]->p % 16 || v[j]->batch % 8 || v[j]->row % 8 || v[j]->head % 8)) return -4;
    if (p.w[i] && (uintptr_t)p.w[i] % 16) return -4;
  }
  return 0;
}
static int qr_blocks_for(const PdtQkRope& p) {  // workgroups that give every wave one step over the tokens
  const int l = qr_lanes(p), per_wave = (64 / l) / qr_groups(p, l);
  return (int)(((int64_t)p.T + QR_WAVES * per_wave - 1) / (QR_WAVES * per_wave));
}

template <typename T, int L>
static int qr_launch(const PdtQkRope& p, bool bwd, float* partial, hipStream_t st) {
  const int gt = qr_groups(p, L), mode = p.R == 0 ? 0 : (p.interleaved ? 2 : 1);
  if (bwd) {
    const dim3 grid(pdt_qk_rope_bwd_blocks(&p), 2);
    if (mode == 0) hipLaunchKernelGGL((qk_rope_bwd_kernel<T, L, 0>), grid, dim3(64 * QR_WAVES), 0, st, p, gt, partial);
    else if (mode == 1) hipLaunchKernelGGL((qk_rope_bwd_kernel<T, L, 1>), grid, dim3(64 * QR_WAVES), 0, st, p, gt, partial);
    else hipLaunchKernelGGL((qk_rope_bwd_kernel<T, L, 2>), grid, dim3(64 * QR_WAVES), 0, st, p, gt, partial);
  } else {
    if ((int64_t)qr_blocks_for(p) * 64 * QR_WAVES > 0xFFFFFFFFll) return -3;  // (a launch counts its threads in 32 bits)
    const dim3 grid(qr_blocks_for(p));
    if (mode == 0) hipLaunchKernelGGL((qk_rope_fwd_kernel<T, L, 0>), grid, dim3(64 * QR_WAVES), 0, st, p, gt);
    else if (mode == 1) hipLaunchKernelGGL((qk_rope_fwd_kernel<T, L, 1>), grid, dim3(64 * QR_WAVES), 0, st, p, gt);
    else hipLaunchKernelGGL((qk_rope_fwd_kernel<T, L, 2>), grid, dim3(64 * QR_WAVES), 0, st, p, gt);
  }
  return (int)hipGetLastError();
}
template <typename T>
static int qr_run(const PdtQkRope& p, bool bwd, float* partial, hipStream_t st) {
  switch (qr_lanes(p)) {
    case 1: return qr_launch<T, 1>(p, bwd, partial, st);
    case 2: return qr_launch<T, 2>(p, bwd, partial, st);
    case 4: return qr_launch<T, 4>(p, bwd, partial, st);
    case 8: return qr_launch<T, 8>(p, bwd, partial, st);
    case 16: return qr_launch<T, 16>(p, bwd, partial, st);
  }
  return -3;
}

}  // namespace pdt

using namespace pdt;

extern "C" int pdt_qk_rope_fwd(int dtype, const PdtQkRope* a, void* stream) {
  if (int e = qr_check(dtype, *a, false)) return e;
  if (a->T == 0) return 0;
  return dtype == PDT_F16 ? qr_run<_Float16>(*a, false, nullptr, (hipStream_t)stream)
                          : qr_run<__bf16>(*a, false, nullptr, (hipStream_t)stream);
}
extern "C" int pdt_qk_rope_bwd_blocks(const PdtQkRope* a) {
  const int n = qr_blocks_for(*a);
  return n < 1 ? 1 : (n > QR_BWD_BLOCKS ? QR_BWD_BLOCKS : n);
}
extern "C" int pdt_qk_rope_bwd(int dtype, const PdtQkRope* a, float* partial, void* stream) {
  if (int e = qr_check(dtype, *a, true)) return e;
  return dtype == PDT_F16 ? qr_run<_Float16>(*a, true, partial, (hipStream_t)stream)
                          : qr_run<__bf16>(*a, true, partial, (hipStream_t)stream);
}
