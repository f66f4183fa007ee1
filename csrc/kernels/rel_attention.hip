// Softmax attention with a learned relative position bias for gfx950: any length, any head dim up to 128 that is a
// multiple of 8, strided or packed rows, key mask with holes, dropout on the probabilities, gradients of q, k, v and of
// the bias table.
//
//   s_ij = scale q_i . k_j + table[bucket(j - i)][h],   p = softmax over the attended keys,   o_i = sum_j p_ij v_j
//   backward: dp = do . v,  ds = p (dp - delta),  delta_i = do_i . o_i,  dq = scale ds k,  dk = scale ds^T q,
//             dv = p^T do,  dtable[t][h] = sum of ds_ij over the batch and all (i, j) with bucket(j - i) = t
//
// The bias depends on (head, j - i) only, and is constant once |j - i| reaches max_distance: every workgroup expands its
// head's column of the table into an LDS array over the near distances, and score tiles that lie completely beyond them
// use one constant.  The array exists in four copies shifted by one element, so that the four consecutive distances of a
// lane's accumulator registers are one aligned 16-byte read whatever the lane's query row is.
//
// The table gradient is the sum of ds along its diagonals.  A 16x16 tile of ds (keys in registers, queries in lanes) is
// reduced to its 31 diagonals with DPP row shifts (register r shifted by r lanes lines the diagonals up) and added to an
// LDS array that belongs to the wave; far tiles only add up their elements.  No two waves share an array and nothing is
// accumulated through global atomics, so the gradient does not depend on the order in which workgroups run.
//
// Products put the key (forward, dQ) or the query (dK / dV) on the register axis, so that an accumulator tile is directly
// the B operand of the next product; rows come through LDS in chunks of 64, double-buffered, filled by LDS-DMA.  A row
// that no query may attend to is read as zeros: whatever its memory holds, NaN included, never meets a product.
//
// P and dS enter the products as 16-bit operands, the one place where something is rounded before the results are.  A second
// operand with what that leaves would make 13 products of a training pass's 9; without it the results are off by 2.4e-3 of their
// norm in bf16 and 2.9e-4 in fp16, where rounding the results alone leaves 1.7e-3 and 2.1e-4.
//
// Measured, forward / dQ / dK and dV (short: one backward kernel), us and the rate of the products that are wanted:
//   1 x 17, 12 heads of 64          6.5                     a launch
//   32 x 128, 16 heads              11.1                    a launch, then waves waiting for their rows
//   256 x 128, 16 heads, fp16       53-63 / 135             memory and its latency: the four and eight arrays once are 104 together
//   32 x 512, 12 heads, bf16        49 / 74 / 69            rounds of workgroups; masks and near tiles in every chunk
//   2 x 4096, 16 heads, bf16        190 / 239 / 266         0.7, 0.85 and 1.0 PFLOP/s: LDS reads, exp2 and products share the issue, and
//                                                           1024 workgroups make a round and a third of the 768 places of the first two
//   1 x 8191, 12 heads, bf16        254 forward             0.82 PFLOP/s, one whole round
//   4 x 1001, 8 heads of 128, holes 39 / 57 / 46            every chunk is masked: tiles read bias and mask from LDS also far out
// With dropout 0.1: 256 x 128 without a mask, fp16 77 / 155 -> 82 / 203, bf16 72 / 142 -> 77 / 178; 32 x 512 51 / 78 / 70 -> 60 / 97 / 83;
// 2 x 4096 188 / 239 / 267 -> 239 / 328 / 352 (a hash and a select per score, and registers that spill, see below).
#include <mutex>
#include <type_traits>
#include <unordered_set>

#include "attn_common.hpp"

namespace pdt {

constexpr int RA_WAVES = 4, RA_THREADS = RA_WAVES * 64;
constexpr int RA_CHUNK = 64;                    // rows per LDS image
constexpr int RA_IMG = RA_CHUNK * 128;          // bytes of a 64-row x 64-column image
constexpr int RA_MAX_FAR = 512;                 // largest max_distance
constexpr int RA_MAX_STEPS = 32;                // logarithmic buckets per side
constexpr float RA_SLACK = 8.0f, RA_SLACK_DROP = 4.0f;  // (with dropout p is divided by the share kept as well)
// Waves per SIMD that the register allocation of a kernel with QB blocks of KS 32-column steps must allow.  At QB KS = 4:
// forward and dQ 3 (dQ with 2: 83 instead of 75 us at 32 x 512 tokens, 12 heads), dK / dV 2 (with 3 86 instead of 73 us).  Three
// waves leave 168 registers, which hold the forward (154) but not all of dQ in its 128-row shape: 9 (fp16) and 10 (bf16) go to
// scratch.  With dropout it spills 14 and 16, the 64-row shape 13 and 11, the forward 2; the 128-row short
// backward, at 128 registers, 23 and 18.  The limits were chosen without dropout.
#define RA_OCC_FWD __attribute__((amdgpu_waves_per_eu(KS * QB <= 4 ? 3 : 2, 8)))
#define RA_OCC_DQ __attribute__((amdgpu_waves_per_eu(KS * QB <= 4 ? 3 : 2, 8)))
#define RA_OCC_DKV __attribute__((amdgpu_waves_per_eu(KS * QB <= 2 ? 3 : 2, 8)))

// rows [0, 64) of a [rows][D] matrix (row stride `stride` elements) into NH 64-column images: 16-byte chunk c of row r is
// stored at chunk c ^ (r & 6).  Rows whose bit in `rows` is clear, and columns from D on, arrive as zeros.  The pieces of a
// wave lie 8 WAVES rows apart (and 64 columns), which goes into the descriptor: one offset per lane serves all of them.
template <typename T, int NH, int WAVES = RA_WAVES>
__device__ __forceinline__ void ra_stage(char* img, const T* src, uint32_t stride, uint64_t rows, int D, int lane, int wave) {
  const int row0 = wave * 8 + (lane >> 3), col0 = ((lane & 7) ^ (row0 & 6)) << 3;
  const uint32_t off = (row0 * stride + col0) * 2u;
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int u = 0; u < 8 / WAVES; ++u) {
      const int first = u * 8 * WAVES;
      const int4v rsrc = pdt_make_rsrc(src + (int64_t)first * stride + h * 64, rows ? (uint32_t)((RA_CHUNK - 1 - first) * stride + D - h * 64) * 2u : 0u);
      const bool ok = ((rows >> (first + row0)) & 1) && col0 + h * 64 < D;
      pdt_lds_dma16(rsrc, img + h * RA_IMG + (u * WAVES + wave) * 1024, ok ? off : 0x80000000u);
    }
  }
}
// rows x0..x0+15 as an A operand: lane -> row x0 + (lane & 15), k = 8 (lane >> 4) + j of the 32-column step ks
__device__ __forceinline__ short8 ra_row_frag(const char* img, int x0, int ks, int lane) {
  const int row = x0 + (lane & 15), c = (ks & 1) * 4 + (lane >> 4);
  return *reinterpret_cast<const short8*>(img + (ks >> 1) * RA_IMG + row * 128 + ((c ^ (row & 6)) << 4));
}
// transposed operand over 32 rows from r0: lane -> column 16 db + (lane & 15); k-value j < 4: row r0 + 4 g + j, j >= 4:
// row r0 + 16 + 4 g + (j - 4) - the order in which pack_pair() lays out two accumulator tiles
__device__ __forceinline__ short8 ra_tr_frag(const char* img, int r0, int db, int lane) {
  const int g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3;
  const int row = r0 + 4 * g + q, c = 2 * (db & 3) + (p >> 1);
  const char* a = img + (db >> 2) * RA_IMG + row * 128 + ((c ^ (row & 6)) << 4) + (p & 1) * 8;
  const short4r lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4r __attribute__((address_space(3)))*)PDT_LDS_PTR(a));
  const short4r hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4r __attribute__((address_space(3)))*)PDT_LDS_PTR(a + 16 * 128));
  return short8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
// the lane's 8 values of a row in global memory (zeros from column D on, or when the row is not there)
template <typename T>
__device__ __forceinline__ short8 ra_gfrag(const T* row, int ks, int D, int lane, bool ok) {
  const int col = ks * 32 + (lane >> 4) * 8;
  short8 r = {0, 0, 0, 0, 0, 0, 0, 0};
  if (ok && col < D) r = *reinterpret_cast<const short8*>(row + col);
  return r;
}
// A wave's 16-row tile t[2 KS] (lane (lm, g) holds row lm, columns 16 db + 4 g + r) as 16-bit rows: lanes g and g ^ 1
// swap a block of every pair, so that each stores 16 contiguous bytes.  Call with the whole wave.
template <typename T, int KS>
__device__ __forceinline__ void ra_store(T* row, const float4v (&t)[2 * KS], float mul, int g, int D, bool valid) {
  const bool odd = g & 1;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    int2v pk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4v v = t[2 * ks + i] * mul;
      pk[i] = int2v{cvt_pk<T>(v[0], v[1]), cvt_pk<T>(v[2], v[3])};
    }
    const int2v own = odd ? pk[1] : pk[0], snd = odd ? pk[0] : pk[1];
    int2v rcv;
    rcv[0] = __shfl_xor(snd[0], 16, 64); rcv[1] = __shfl_xor(snd[1], 16, 64);
    const int col = ks * 32 + (odd ? 16 : 0) + 4 * (g & ~1);
    if (valid && col < D)
      *reinterpret_cast<int4v*>(row + col) = odd ? int4v{rcv[0], rcv[1], own[0], own[1]} : int4v{own[0], own[1], rcv[0], rcv[1]};
  }
}

// maximum / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48) with register swaps instead of LDS permutes
__device__ __forceinline__ float ra_other16(float v, float& mine) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  mine = __uint_as_float(r[0]);
  return __uint_as_float(r[1]);
}
__device__ __forceinline__ float ra_other32(float v, float& mine) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  mine = __uint_as_float(r[0]);
  return __uint_as_float(r[1]);
}
__device__ __forceinline__ float ra_quad_max(float v) {
  float a, b = ra_other16(v, a);
  v = fmaxf(a, b);
  b = ra_other32(v, a);
  return fmaxf(a, b);
}
__device__ __forceinline__ float ra_quad_sum(float v) {
  float a, b = ra_other16(v, a);
  v = a + b;
  b = ra_other32(v, a);
  return a + b;
}

// ---- the lift of an fp16 backward pass
// P and ds are operands of 16 bits.  ds has the size of P times the output gradients, 1e-7 for 1000 keys and gradients of 1e-4,
// and as it stands fp16 would round it to steps of 6e-8 (1000 keys, gradients of 1e-4: an error of 9.9e-3 of dQ, where relative
// roundings leave 5.1e-4; 2100 keys and 1e-3: 2.2e-3 and 4.1e-4).  So P enters the products as 2^lift P, with the power of two that brings the largest |dout| of
// the rows that share it to [1/2, 1), and the results are multiplied by 2^-lift: the factor rides on the exponent of P and on
// final scales that are there anyway.  2^lift P over the share kept stays below 2^15; |ds| 2^lift stays below what output
// gradients of size one give without a lift, half the sum of |v| over a row (p (1 - p) times the spread of dp) but for
// dropout's factor.  bf16 has fp32's exponents: no lift.  Backward of 256 x 128 tokens, 16 heads: 150 -> 152 us, with dropout 184 ->
// 197 (five more registers spill); of 2 x 4096 tokens no difference.
template <typename T> constexpr bool RA_LIFTS = std::is_same<T, _Float16>::value;
// the largest of the bits of |x| over eight 16-bit values (ordered like the values; infinities and NaN are larger than all numbers)
__device__ __forceinline__ uint32_t ra_top(uint32_t top, const short8& x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, (uint32_t)x[j] & 0x7FFFu);
  return top;
}
template <int CTRL>
__device__ __forceinline__ uint32_t ra_ror_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t ra_wave_max(uint32_t v) {  // (wave-uniform; no LDS permutes, whose addresses would stay in registers)
  v = ra_ror_max<0x121>(ra_ror_max<0x122>(ra_ror_max<0x124>(ra_ror_max<0x128>(v))));  // row_ror:8, 4, 2, 1
  const auto at = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
  return max(max(at(0), at(16)), max(at(32), at(48)));
}
__device__ __forceinline__ int ra_lift(uint32_t top, float drop_scale) {
  const int room = 14 - ((int)(__float_as_uint(drop_scale) >> 23) - 127);  // (the share kept: at most 2^room / 2^15)
  return min(max(14 - (int)(top >> 10), 0), room);
}

// ---- one (batch, head) of a launch
struct RaSpan {
  int b, h, n;      // sample, head, length
  int64_t row0;     // first packed row (packed) or 0
};
__device__ __forceinline__ RaSpan ra_span(const PdtRelAttn& p, int bh) {
  RaSpan s;
  s.b = bh / p.A;
  s.h = bh - s.b * p.A;
  if (p.cu) {  // (lengths that do not fit the tensors are cut to them)
    const int lo = min(max(uniform_load_i32(p.cu, s.b), 0), p.T), hi = min(max(uniform_load_i32(p.cu, s.b + 1), lo), p.T);
    s.row0 = lo;
    s.n = min(hi - lo, p.S);
  } else {
    s.row0 = 0;
    s.n = p.S;
  }
  return s;
}
template <typename T>
__device__ __forceinline__ T* ra_base(const PdtRelView& v, const RaSpan& s, bool packed) {
  return (T*)v.p + (packed ? s.row0 * v.row : (int64_t)s.b * v.batch) + (int64_t)s.h * v.head;
}
// Rows of a packed output that no sample takes in become zero: those from cu[B] on (by the last sample's workgroups), those
// before cu[0] (by the first's) and what of a sample lies beyond the longest length announced (by its own).
template <typename T>
__device__ __forceinline__ void ra_tail(const PdtRelAttn& p, const RaSpan& s, const PdtRelView& v, int tid, int threads) {
  if (!p.cu) return;
  const int per = p.D >> 3;
  auto zero = [&](int64_t first, int64_t end) {
    const int64_t n = (end - first) * per;
    for (int64_t i = (int64_t)blockIdx.y * threads + tid; i < n; i += (int64_t)gridDim.y * threads) {
      const int64_t r = i / per, c = i - r * per;
      *reinterpret_cast<int4v*>((T*)v.p + (first + r) * v.row + (int64_t)s.h * v.head + c * 8) = int4v{0, 0, 0, 0};
    }
  };
  zero(s.row0 + s.n, s.b == p.B - 1 ? p.T : min(max(uniform_load_i32(p.cu, s.b + 1), 0), p.T));
  if (s.b == 0) zero(0, s.row0);
}
// attended keys of chunk c, one bit each
__device__ __forceinline__ uint64_t ra_word(const PdtRelAttn& p, const RaSpan& s, int c) {
  const int left = s.n - c * RA_CHUNK;
  if (left <= 0) return 0;
  uint64_t w = left >= RA_CHUNK ? ~0ull : (1ull << left) - 1;
  if (p.mask) {  // (the whole wave comes here together)
    const int k = c * RA_CHUNK + (threadIdx.x & 63);
    const int64_t at = (int64_t)s.b * p.mask_stride + k;
    bool on = false;
    if (k < s.n) on = p.mask_bytes == 1 ? ((const uint8_t*)p.mask)[at] != 0 : ((const int32_t*)p.mask)[at] != 0;
    w &= __ballot(on);
  }
  if (p.mask_bits) w &= ((const __attribute__((address_space(4))) uint64_t*)p.mask_bits)[(int64_t)s.b * p.mask_words + c];
  return w;
}
// The chunks of a sweep that hold an attended row, in ascending order.  Whole chunks (every row attended) beyond the near
// distances have one bias, whole near ones look theirs up, the others mask rows as well: runs of each kind take turns in
// three loops with one form of the score arithmetic each.  The forms as branches of one loop cost 45 to 85 registers more, and
// a wave of occupancy with them.
enum { RA_FARAWAY, RA_NEAR, RA_PARTIAL };
template <int K> using RaKind = std::integral_constant<int, K>;
struct RaChunks {
  int c, nc, lo, hi;  // current chunk; far chunks lie at or below lo or at or above hi
  int buf;            // the LDS buffer it is staged in
  uint64_t w;         // its attended rows
  template <typename WordFn>
  __device__ __forceinline__ void next(WordFn word) {
    for (++c; c < nc; ++c)
      if ((w = word(c)) != 0) break;
  }
  __device__ __forceinline__ bool done() const { return c >= nc; }
  __device__ __forceinline__ int kind() const { return w != ~0ull ? RA_PARTIAL : (c <= lo || c >= hi ? RA_FARAWAY : RA_NEAR); }
};
// `rows` rows from w0 on against chunks of 64: a chunk is far when all its tiles lie at least `far` beyond all rows
__device__ __forceinline__ RaChunks ra_chunks(int n, int w0, int rows, int far, bool has_bias) {
  RaChunks k;
  k.nc = (n + RA_CHUNK - 1) / RA_CHUNK;
  // 64 c + 48 - w0 <= -(far + 16)   and   64 c - (w0 + rows - 16) >= far + 16
  k.lo = w0 - far >= RA_CHUNK ? (w0 - far) / RA_CHUNK - 1 : -1;
  k.hi = (w0 + rows + far + RA_CHUNK - 1) / RA_CHUNK;
  if (!has_bias) k.lo = k.nc;
  k.c = -1;
  k.buf = 0;
  k.w = 0;
  return k;
}

// ---- the bias array: entry i of copy j is the bias (times log2 e, `plus` a constant) of distance sign * (i + j - off); `off`
// and the clamp leave room so that a tile beyond the near distances reads the constant part.
struct RaBias {
  float* t;
  int len, off, far;  // far: max_distance rounded up to the tile size
};
__device__ __forceinline__ int ra_far(int max_distance) { return (max_distance + 15) & ~15; }
__host__ __device__ inline int ra_bias_len(int max_distance) {
  const int n = 2 * ((max_distance + 15) & ~15) + 64;
  return (n - 16 + 63) / 64 * 64 + 16;  // the copies start 64 bytes apart modulo the 256 bytes of one access
}
__host__ __device__ inline int ra_diag_len(int max_distance) { return 2 * ((max_distance + 15) & ~15) + 64; }
__device__ __forceinline__ int ra_bucket(const PdtRelAttn& p, int d) {
  const int n = d < 0 ? -d : d, half = p.buckets >> 1, exact = half >> 1;
  int b = n;
  if (n >= exact) {
    b = exact;
    for (int j0 = 1; j0 < half - exact; j0 += 8) {  // (eight at a time: one scalar load; the entries behind the last are INT_MAX)
#pragma unroll
      for (int j = 0; j < 8; ++j) b += n >= p.steps[j0 + j] ? 1 : 0;
    }
  }
  return b + (d > 0 ? half : 0);
}
template <typename T>
__device__ __forceinline__ float ra_table(const PdtRelAttn& p, int bucket, int h) {
  const int64_t i = (int64_t)bucket * p.A + h;
  return p.table_f32 ? ((const float*)p.table)[i] : Half16<T>::to_f(((const short*)p.table)[i]);
}
template <typename T, int THREADS = RA_THREADS>
__device__ __forceinline__ RaBias ra_bias_fill(const PdtRelAttn& p, float* mem, int h, int sign, int tid, int max_distance, float plus = 0.f) {
  RaBias t{mem, ra_bias_len(max_distance), ra_far(max_distance) + 32, ra_far(max_distance)};
  for (int i = tid; i < t.len + 4; i += THREADS) {
    const float v = (p.table ? ra_table<T>(p, ra_bucket(p, sign * (i - t.off)), h) * LOG2E : 0.f) + plus;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i - j >= 0 && i - j < t.len) mem[j * t.len + i - j] = v;
  }
  return t;
}
// the lane's offset into the array: distances u + 4 g + r - lm (r = 0..3) of a tile u apart start at t[lane_off + u]
__device__ __forceinline__ int ra_bias_lane(const RaBias& t, int lm, int g) {
  const int j = -lm & 3;
  return j * t.len + t.off + 4 * g - lm - j;
}
__device__ __forceinline__ float4v ra_bias4(const RaBias& t, int lane_off, int u) {
  const int uc = min(max(u, -(t.far + 16)), t.far + 16);
  return *reinterpret_cast<const float4v*>(t.t + lane_off + uc);
}

// ------------------------------------------------------------------------------------------------ forward
// One wave = 16 QB query rows against all keys, or (SPLIT 2) against half of every chunk; online softmax in the log2 domain.
template <typename T, int KS, int QB, int SPLIT, bool DROP>
__global__ __launch_bounds__(RA_THREADS) RA_OCC_FWD void rel_attn_fwd_kernel(PdtRelAttn p) {
  constexpr int NH = (KS + 1) / 2, BUF = 2 * NH * RA_IMG;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, lm = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RaSpan s = ra_span(p, blockIdx.x);
  constexpr int ROWS = RA_WAVES / SPLIT * 16 * QB;
  const int group = SPLIT == 2 ? wave & 1 : wave, half = SPLIT == 2 ? wave >> 1 : 0;
  const int w0 = blockIdx.y * ROWS, q0 = w0 + group * 16 * QB;
  ra_tail<T>(p, s, p.o, tid, RA_THREADS);
  if (w0 >= s.n) return;
  const bool packed = p.cu != nullptr;
  const T* qb_ = ra_base<const T>(p.q, s, packed);
  const T* kb_ = ra_base<const T>(p.k, s, packed);
  const T* vb_ = ra_base<const T>(p.v, s, packed);
  float* const mb = reinterpret_cast<float*>(smem + 2 * BUF);  // 0 / -inf of the 64 keys of each buffer
  auto stage = [&](int c, int buf, uint64_t w) {
    char* m = smem + buf * BUF;
    ra_stage<T, NH>(m, kb_ + (int64_t)c * RA_CHUNK * p.k.row, (uint32_t)p.k.row, w, p.D, lane, wave);
    ra_stage<T, NH>(m + NH * RA_IMG, vb_ + (int64_t)c * RA_CHUNK * p.v.row, (uint32_t)p.v.row, w, p.D, lane, wave);
    if (tid < RA_CHUNK) mb[buf * RA_CHUNK + tid] = (w >> tid) & 1 ? 0.f : -INFINITY;
  };
  auto word = [&](int c) { return ra_word(p, s, c); };
  const float k2 = p.scale * LOG2E;
  RaChunks cur = ra_chunks(s.n, w0, ROWS, ra_far(p.max_distance), p.table != nullptr);
  cur.next(word);
  const bool active = q0 < s.n;
  short8 qf[QB][KS];
#pragma unroll
  for (int i = 0; i < QB; ++i)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[i][ks] = ra_gfrag<T>(qb_ + (int64_t)(q0 + 16 * i + lm) * p.q.row, ks, p.D, lane, q0 + 16 * i + lm < s.n);
  if (!cur.done()) stage(cur.c, 0, cur.w);
  const RaBias bias = ra_bias_fill<T>(p, mb + 2 * RA_CHUNK, s.h, 1, tid, p.max_distance);
  const int boff = ra_bias_lane(bias, lm, g);
  uint32_t seed[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i)
    seed[i] = DROP ? attn_row_seed(drop_key(p.rng), drop_sample(p.rng, s.b) * p.A + s.h, q0 + 16 * i + lm) : 0u;
  const uint32_t thr_hi = attn_thr_hi(p.drop_thr), kmul0 = (uint32_t)(4 * g) * ATT_GOLD;
  // Running maximum m of a row (log2 domain), and what the products start from: c0 = -m / k2, so that the scores come out of
  // the matrix unit with the maximum subtracted.  m = -inf: no attended key so far (the products then start from 0).
  const float inv_k2 = 1.0f / k2;
  constexpr int ZONE = RA_WAVES * 16 * QB;
  float* const zone = bias.t + 4 * bias.len + wave * 16 * QB + lm;  // [2][ZONE]: log2 of the rows' sums at the near chunks' ends
  float m[QB];
  float4v c0[QB], l4[QB], o[QB][2 * KS];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    m[i] = -INFINITY;
    c0[i] = l4[i] = splat4(0.f);
#pragma unroll
    for (int db = 0; db < 2 * KS; ++db) o[i][db] = splat4(0.f);
  }
  __syncthreads();  // the bias array is complete
  const float bias_lo = bias.t[0], bias_hi = bias.t[bias.len - 1];
  auto sweep = [&](auto kind, RaChunks cur, int stop) {
    constexpr int KIND = decltype(kind)::value;
    constexpr float SLACK = DROP ? RA_SLACK_DROP : RA_SLACK;
    while (cur.c < stop && cur.kind() == KIND) {
      const int buf = cur.buf;
      RaChunks nx = cur;
      nx.next(word);
      nx.buf ^= 1;
      __syncthreads();  // every wave is done with the other buffer
      if (!nx.done()) {
        stage(nx.c, buf ^ 1, nx.w);
        if (NH == 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __syncthreads();
      if (active) {
        const char* kimg = smem + buf * BUF;
        const char* vimg = kimg + NH * RA_IMG;
        const int u0 = cur.c * RA_CHUNK - q0;
        const float flat = cur.c <= cur.lo ? bias_lo : bias_hi;
#pragma unroll
        for (int pi = 0; pi < 2 / SPLIT; ++pi) {  // 32 keys at a time
          const int pb = SPLIT == 2 ? half : pi;
          float4v sc[QB][2];
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
#pragma unroll
            for (int i = 0; i < QB; ++i) sc[i][hb] = c0[i];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const short8 kf = ra_row_frag(kimg, pb * 32 + hb * 16, ks, lane);
#pragma unroll
              for (int i = 0; i < QB; ++i) sc[i][hb] = Half16<T>::mfma(kf, qf[i][ks], sc[i][hb]);
            }
          }
          short8 pf[QB];
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            float cmax = -INFINITY;
#pragma unroll
            for (int hb = 0; hb < 2; ++hb) {
              const int k16 = pb * 32 + hb * 16;
              float4v b = splat4(flat);
              if (KIND != RA_FARAWAY) b = ra_bias4(bias, boff, u0 + k16 - 16 * i);
              if (KIND == RA_PARTIAL) b += *reinterpret_cast<const float4v*>(mb + buf * RA_CHUNK + k16 + 4 * g);
              const float4v t = sc[i][hb] * k2 + b;
              cmax = fmaxf(fmaxf(cmax, t[0]), fmaxf(fmaxf(t[1], t[2]), t[3]));
              sc[i][hb] = t;
            }
            // The accumulators are rescaled only when some row's maximum has grown by more than 2^SLACK since its last
            // rescale: p then stays below 2^SLACK instead of 1, which 16-bit operands and fp32 sums hold as exactly.
            if (__any(cmax > (m[i] == -INFINITY ? -INFINITY : SLACK))) {
              const float used = m[i] == -INFINITY ? 0.f : m[i], m_new = fmaxf(m[i], ra_quad_max(cmax) + used);
              const float now = m_new == -INFINITY ? 0.f : m_new;
              const float alpha = __builtin_amdgcn_exp2f(m[i] - now);
              m[i] = m_new;
              c0[i] = splat4(-now * inv_k2);
              sc[i][0] += used - now;
              sc[i][1] += used - now;
              l4[i] *= alpha;
#pragma unroll
              for (int db = 0; db < 2 * KS; ++db) o[i][db] *= alpha;
            }
#pragma unroll
            for (int hb = 0; hb < 2; ++hb) {
              float4v t = sc[i][hb];
#pragma unroll
              for (int r = 0; r < 4; ++r) t[r] = __builtin_amdgcn_exp2f(t[r]);
              l4[i] += t;
              if (DROP) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  t[r] *= attn_keep(seed[i], kmul0 + (uint32_t)(cur.c * RA_CHUNK + pb * 32 + hb * 16 + r) * ATT_GOLD, thr_hi) ? p.drop_scale : 0.f;
              }
              sc[i][hb] = t;
            }
            pf[i] = pack_pair<T>(sc[i][0], sc[i][1]);
          }
#pragma unroll
          for (int db = 0; db < 2 * KS; ++db) {
            const short8 vf = ra_tr_frag(vimg, pb * 32, db, lane);
#pragma unroll
            for (int i = 0; i < QB; ++i) o[i][db] = Half16<T>::mfma(vf, pf[i], o[i][db]);
          }
        }
      }
      cur = nx;
    }
    return cur;
  };
#pragma unroll 1
  for (int z = 0; z < 3; ++z) {  // the chunks below the near ones, the near ones, those above
    const int stop = p.mass && z < 2 ? min(z ? cur.hi : cur.lo + 1, cur.nc) : cur.nc;
    while (cur.c < stop)
      cur = sweep(RaKind<RA_PARTIAL>{}, sweep(RaKind<RA_NEAR>{}, sweep(RaKind<RA_FARAWAY>{}, cur, stop), stop), stop);
    if (!p.mass) break;
    if (z == 2) break;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const float t = ra_quad_sum((l4[i][0] + l4[i][1]) + (l4[i][2] + l4[i][3]));
      if (g == 0) zone[z * ZONE + 16 * i] = m[i] + __log2f(t);  // (-inf where nothing was summed)
    }
  }
  float l[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) l[i] = (l4[i][0] + l4[i][1]) + (l4[i][2] + l4[i][3]);
  if (SPLIT == 2) {  // the two waves of a row group join their halves of the keys
    constexpr int F = QB * (8 * KS + 2);
    static_assert(2 * F * 64 * (int)sizeof(float) <= 2 * BUF, "the join reuses the images");
    float* x = reinterpret_cast<float*>(smem) + group * F * 64 + lane;
    __syncthreads();
    if (half == 1 && active) {
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        float* y = x + i * (8 * KS + 2) * 64;
#pragma unroll
        for (int e = 0; e < 8 * KS; ++e) y[e * 64] = o[i][e >> 2][e & 3];
        y[8 * KS * 64] = m[i];
        y[(8 * KS + 1) * 64] = l[i];
      }
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const float* y = x + i * (8 * KS + 2) * 64;
      if (!active) break;
      const float m2 = y[8 * KS * 64], top = fmaxf(m[i], m2), use = top == -INFINITY ? 0.f : top;
      const float a = __builtin_amdgcn_exp2f(m[i] - use), b = __builtin_amdgcn_exp2f(m2 - use);
      m[i] = top;
      l[i] = l[i] * a + y[(8 * KS + 1) * 64] * b;
#pragma unroll
      for (int e = 0; e < 8 * KS; ++e) o[i][e >> 2][e & 3] = o[i][e >> 2][e & 3] * a + y[e * 64] * b;
    }
  }
  if (!active) return;
  T* ob = ra_base<T>(p.o, s, packed);
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = q0 + 16 * i + lm;
    const float total = ra_quad_sum(l[i]);
    // a row without an attended key has no probability mass: a zero output, and lse = +inf makes every p of backward 0
    // (the sum is NaN, not 0, when a score was: the output is then NaN as well)
    const int64_t row = ((int64_t)s.b * p.A + s.h) * p.S + q;
    const float lse = total == 0.f ? INFINITY : m[i] + __log2f(total);
    if (p.lse && g == 0 && q < s.n) p.lse[row] = lse;
    if (p.mass && g == 0 && q < s.n) {
      float lo = __builtin_amdgcn_exp2f(zone[16 * i] - lse), in = __builtin_amdgcn_exp2f(zone[ZONE + 16 * i] - lse);
      if (SPLIT == 2) {
        lo += __builtin_amdgcn_exp2f(zone[16 * (i + 2 * QB)] - lse);
        in += __builtin_amdgcn_exp2f(zone[ZONE + 16 * (i + 2 * QB)] - lse);
      }
      p.mass[row] = cur.lo < 0 ? 0.f : lo;
      p.mass[(int64_t)p.B * p.A * p.S + row] = cur.hi >= cur.nc || 1.f - in < 0x1p-16f ? 0.f : 1.f - in;  // (less is the rounding of `in`)
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    ra_store<T, KS>(ob + (int64_t)q * p.o.row, o[i], inv, g, p.D, q < s.n);
    if (p.o_lo.p) {
#pragma unroll
      for (int db = 0; db < 2 * KS; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = o[i][db][r] * inv;
          o[i][db][r] = v - Half16<T>::to_f(Half16<T>::from_f(v));
        }
      ra_store<T, KS>(ra_base<T>(p.o_lo, s, packed) + (int64_t)q * p.o_lo.row, o[i], 1.0f, g, p.D, q < s.n);
    }
  }
}

// Sums of ds along its diagonals, from 16x16 tiles (lane (lm, g): keys 4 g + r, query lm) of blocks u apart:
// N: lane l holds the sum over r of the elements at (4 g + r, l + r), distance u + 4 g - l.  W: those with l + r >= 16, i.e.
// query l + r - 16, distance u + 4 g - l + 16 (lanes 13..15 only): the place that N of the tile at u + 16 has in the same lane.
__device__ __forceinline__ float ra_diag_n(const float4v& t) {
  float n = t[0];
  n += dpp_f<0x101>(t[1]);  // row_shl:1
  n += dpp_f<0x102>(t[2]);
  n += dpp_f<0x103>(t[3]);
  return n;
}
__device__ __forceinline__ float ra_diag_w(const float4v& t) {
  float w = dpp_f<0x11F>(t[1]);  // row_shr:15
  w += dpp_f<0x11E>(t[2]);
  w += dpp_f<0x11D>(t[3]);
  return w;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float ra_dpp_rows(float old, float v) {  // the rows in ROWS shifted (zeros come in), the others from old
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xF, true));
}
// N summed over the lane groups, whose distances are 4 lanes apart: place l' = l + 12 - 4 g has distance u + 12 - l'.  Lanes
// 0..31 receive the places 0..15 (each twice), lanes 32..63 the places 16..27 (and four zeros).
__device__ __forceinline__ float ra_diag_fold(float n) {
  float low = ra_dpp_rows<0x11C, 1>(n, n);  // row_shr:12 of group 0
  low = ra_dpp_rows<0x118, 2>(low, n);
  low = ra_dpp_rows<0x114, 4>(low, n);
  float high = ra_dpp_rows<0x104, 1>(0.f, n);  // what left the row: row_shl:4 of group 0
  high = ra_dpp_rows<0x108, 2>(high, n);
  high = ra_dpp_rows<0x10C, 4>(high, n);
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(low), __float_as_uint(high), false, false);
  float a, b = ra_other16(__uint_as_float(r[0]) + __uint_as_float(r[1]), a);
  return a + b;
}
// The diagonal sums of one wave.  Tiles arrive in ascending order of u; each near u stores its places once (two arrays: places
// 0..15 and 16..27 of different u fall on the same distances) and hands W to the next.  LDS float atomics instead of this cost
// 24 us of 134 at 32 x 512 tokens, 12 heads, and four times the arrays.
struct RaDiag {
  float* at;    // where this lane stores for u = 0
  float w;
  int u;        // the last near tile (a multiple of 16), or NONE
  static constexpr int NONE = -(1 << 20);
  __device__ __forceinline__ void store(int v, float n) { at[v] = ra_diag_fold(n); }
  __device__ __forceinline__ void flush() {
    if (u != NONE) store(u + 16, w);
    u = NONE;
  }
  __device__ __forceinline__ void add(int v, const float4v& t) {
    if (u != NONE && u + 16 != v) flush();
    store(v, ra_diag_n(t) + (u != NONE ? w : 0.f));
    w = ra_diag_w(t);
    u = v;
  }
};

template <int N>
__device__ __forceinline__ float ra_sum(const float (&v)[N]) {
  float s = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) s += v[i];
  return s;
}

// distances -> buckets: sums[top + d] is the sum at distance d, |d| <= top; eight lanes per bucket walk its range
template <int THREADS>
__device__ __forceinline__ void ra_bucket_sums(const PdtRelAttn& p, const float* sums, int top, float* part, int tid) {
  const int half = p.buckets >> 1, exact = half >> 1;
  for (int b0 = 0; b0 < p.buckets; b0 += THREADS / 8) {
    const int b = b0 + (tid >> 3), j = b >= half ? b - half : b;
    float sum = 0.f;
    if (b < p.buckets) {
      int lo = j < exact ? j : p.steps[j - exact], hi = j < exact ? j : (j == half - 1 ? top : p.steps[j + 1 - exact] - 1);
      if (b >= half) lo = max(lo, 1);
      hi = min(hi, top);
      for (int n = lo + (tid & 7); n <= hi; n += 8) sum += sums[(b >= half ? n : -n) + top];
    }
    sum += __shfl_xor(sum, 1, 64);
    sum += __shfl_xor(sum, 2, 64);
    sum += __shfl_xor(sum, 4, 64);
    if (b < p.buckets && (tid & 7) == 0) part[(int64_t)b * p.A] = sum;
  }
}

// ------------------------------------------------------------------------------------------------ dQ and the table gradient
// One wave = 16 QB query rows, sweeps the keys (SPLIT 2: half of every chunk); also stores delta = rowsum(dO * O) for the dK / dV kernel.
template <typename T, int KS, int QB, int SPLIT, bool DROP>
__global__ __launch_bounds__(RA_THREADS) RA_OCC_DQ void rel_attn_dq_kernel(PdtRelAttn p) {
  constexpr int NH = (KS + 1) / 2, BUF = 2 * NH * RA_IMG;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, lm = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RaSpan s = ra_span(p, blockIdx.x);
  constexpr int ROWS = RA_WAVES / SPLIT * 16 * QB;
  const int group = SPLIT == 2 ? wave & 1 : wave, half = SPLIT == 2 ? wave >> 1 : 0;
  const int w0 = blockIdx.y * ROWS, q0 = w0 + group * 16 * QB;
  float* part = p.dtable_part ? p.dtable_part + ((int64_t)s.b * gridDim.y + blockIdx.y) * p.buckets * p.A + s.h : nullptr;
  ra_tail<T>(p, s, p.dq, tid, RA_THREADS);
  if (w0 >= s.n) {
    if (part)
      for (int i = tid; i < p.buckets; i += RA_THREADS) part[(int64_t)i * p.A] = 0.f;
    return;
  }
  const bool packed = p.cu != nullptr;
  const T* qb_ = ra_base<const T>(p.q, s, packed);
  const T* kb_ = ra_base<const T>(p.k, s, packed);
  const T* vb_ = ra_base<const T>(p.v, s, packed);
  const T* ob_ = ra_base<const T>(p.o, s, packed);
  const T* lb_ = ra_base<const T>(p.o_lo, s, packed);
  const T* gb_ = ra_base<const T>(p.dout, s, packed);
  float* const mb = reinterpret_cast<float*>(smem + 2 * BUF);  // 0 / -inf of the 64 keys of each buffer
  auto stage = [&](int c, int buf, uint64_t w) {
    char* m = smem + buf * BUF;
    ra_stage<T, NH>(m, kb_ + (int64_t)c * RA_CHUNK * p.k.row, (uint32_t)p.k.row, w, p.D, lane, wave);
    ra_stage<T, NH>(m + NH * RA_IMG, vb_ + (int64_t)c * RA_CHUNK * p.v.row, (uint32_t)p.v.row, w, p.D, lane, wave);
    if (tid < RA_CHUNK) mb[buf * RA_CHUNK + tid] = (w >> tid) & 1 ? 0.f : -INFINITY;
  };
  auto word = [&](int c) { return ra_word(p, s, c); };
  RaChunks cur = ra_chunks(s.n, w0, ROWS, ra_far(p.max_distance), p.table != nullptr);
  cur.next(word);
  const bool active = q0 < s.n;
  const int64_t bh = (int64_t)s.b * p.A + s.h;
  short8 qf[QB][KS], df[QB][KS], of[QB][KS], lf[QB][KS];
  const float k2 = p.scale * LOG2E;
  float nlse[QB], nd[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = q0 + 16 * i + lm;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[i][ks] = ra_gfrag<T>(qb_ + (int64_t)q * p.q.row, ks, p.D, lane, q < s.n);
      df[i][ks] = ra_gfrag<T>(gb_ + (int64_t)q * p.dout.row, ks, p.D, lane, q < s.n);
      of[i][ks] = ra_gfrag<T>(ob_ + (int64_t)q * p.o.row, ks, p.D, lane, q < s.n);
      lf[i][ks] = ra_gfrag<T>(lb_ + (int64_t)q * p.o_lo.row, ks, p.D, lane, q < s.n && p.o_lo.p);
    }
    // what the products start from, so that scores come out with lse subtracted (rows that are not there: p = 0)
    nlse[i] = (q < s.n ? -p.lse[bh * p.S + q] : -INFINITY) / k2;
  }
  int lift = 0;  // (of the wave's own rows)
  if constexpr (RA_LIFTS<T>) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) top = ra_top(top, df[i][ks]);
    top = ra_wave_max(top);
    lift = ra_lift(top, p.drop_scale);
    // for the dK / dV kernel, whose sums run over all rows (two waves of a pair hold the same rows and write the same)
    if (lane == 0) p.peaks[(bh * gridDim.y + blockIdx.y) * RA_WAVES + wave] = top;
  }
  const float drop_lift = RA_LIFTS<T> ? __uint_as_float((uint32_t)(127 - lift) << 23) : 1.0f;  // 2^-lift
  if (!cur.done()) stage(cur.c, 0, cur.w);
  const RaBias bias = ra_bias_fill<T>(p, mb + 2 * RA_CHUNK, s.h, 1, tid, p.max_distance);
  const int boff = ra_bias_lane(bias, lm, g);
  // diagonal sums, two arrays per wave: entry 0 is distance -(far + 31)
  const int dlen = ra_diag_len(p.max_distance);
  float* const sums = bias.t + 4 * bias.len;
  RaDiag diag{sums + (wave * 2 + (g >> 1)) * dlen + bias.far + 31 + (g >> 1 ? -4 : 12) - lm, 0.f, RaDiag::NONE};
  if (part)
    for (int i = tid; i < 2 * RA_WAVES * dlen; i += RA_THREADS) sums[i] = 0.f;
  float4v open = splat4(0.f);  // the tile of the last offset, which the next pair of tiles adds to (two blocks per wave)
  int open_u = RaDiag::NONE;
  // A row's ds add up to 0 but for the roundings that its output carries.  Most distances of a long sequence fall into the two
  // far buckets, where ds nearly cancels and these remainders would show (2 x 4096 tokens: 3.3e-3 of the table gradient, now
  // 2.4e-3, for 239 -> 247 us).  The remainder e is what delta is off by, so far sums give back e times their share of the row
  // (p.mass: chunks that are far as a whole; the far tiles of a row's near chunks keep theirs).
  float far_lo = 0.f, far_hi = 0.f, e_all[QB];
  uint32_t seed[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = q0 + 16 * i + lm;
    float d = e_all[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        d += Half16<T>::to_f(df[i][ks][j]) * (Half16<T>::to_f(of[i][ks][j]) + Half16<T>::to_f(lf[i][ks][j]));
    d = ra_quad_sum(d);
    nd[i] = -d;
    if (half == 0 && g == 0 && q < s.n) {  // (for the dK / dV kernel)
      p.delta[bh * p.S + q] = -d;
      p.delta[((int64_t)p.B * p.A + bh) * p.S + q] = nlse[i];
    }
    if (RA_LIFTS<T>) nlse[i] += lift / k2;
    seed[i] = DROP ? attn_row_seed(drop_key(p.rng), drop_sample(p.rng, s.b) * p.A + s.h, q) : 0u;
  }
  const uint32_t thr_hi = attn_thr_hi(p.drop_thr), kmul0 = (uint32_t)(4 * g) * ATT_GOLD;
  float4v dq[QB][2 * KS];
#pragma unroll
  for (int i = 0; i < QB; ++i)
#pragma unroll
    for (int db = 0; db < 2 * KS; ++db) dq[i][db] = splat4(0.f);
  __syncthreads();  // the arrays are complete
  const float bias_lo = bias.t[0], bias_hi = bias.t[bias.len - 1];
  auto near = [&](int u, const float4v& t) {  // (a chunk that is not far may hold far tiles)
    if (u >= bias.far + 16) far_hi += (t[0] + t[1]) + (t[2] + t[3]);
    else if (u <= -(bias.far + 16)) far_lo += (t[0] + t[1]) + (t[2] + t[3]);
    else diag.add(u, t);
  };
  auto sweep = [&](auto kind, RaChunks cur) {
    constexpr int KIND = decltype(kind)::value;
    const bool below = cur.c <= cur.lo;  // (a run of far chunks stays on one side)
    const float before = ra_sum(e_all);
    while (!cur.done() && cur.kind() == KIND && (KIND != RA_FARAWAY || (cur.c <= cur.lo) == below)) {
      const int buf = cur.buf;
      RaChunks nx = cur;
      nx.next(word);
      nx.buf ^= 1;
      __syncthreads();  // every wave is done with the other buffer
      if (!nx.done()) {
        stage(nx.c, buf ^ 1, nx.w);
        if (NH == 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      __syncthreads();
      if (active) {
        const char* kimg = smem + buf * BUF;
        const char* vimg = kimg + NH * RA_IMG;
        const int u0 = cur.c * RA_CHUNK - q0;
#pragma unroll
        for (int pi = 0; pi < 2 / SPLIT; ++pi) {
          const int pb = SPLIT == 2 ? half : pi;
          float4v ds[QB][2];
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            const int k16 = pb * 32 + hb * 16;
            float4v sc[QB], dp[QB];
#pragma unroll
            for (int i = 0; i < QB; ++i) { sc[i] = splat4(nlse[i]); dp[i] = splat4(DROP ? 0.f : nd[i]); }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const short8 kf = ra_row_frag(kimg, k16, ks, lane), vf = ra_row_frag(vimg, k16, ks, lane);
#pragma unroll
              for (int i = 0; i < QB; ++i) {
                sc[i] = Half16<T>::mfma(kf, qf[i][ks], sc[i]);
                dp[i] = Half16<T>::mfma(vf, df[i][ks], dp[i]);
              }
            }
#pragma unroll
            for (int i = 0; i < QB; ++i) {
              float4v b = splat4(below ? bias_lo : bias_hi);
              if (KIND != RA_FARAWAY) b = ra_bias4(bias, boff, u0 + k16 - 16 * i);
              if (KIND == RA_PARTIAL) b += *reinterpret_cast<const float4v*>(mb + buf * RA_CHUNK + k16 + 4 * g);
              float4v t = sc[i] * k2 + b;
#pragma unroll
              for (int r = 0; r < 4; ++r) t[r] = __builtin_amdgcn_exp2f(t[r]);
              float4v e = dp[i];
              if (DROP) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  e[r] *= attn_keep(seed[i], kmul0 + (uint32_t)(cur.c * RA_CHUNK + k16 + r) * ATT_GOLD, thr_hi) ? p.drop_scale : 0.f;
              }
              ds[i][hb] = DROP ? t * (e + nd[i]) : t * e;
            }
          }
          short8 sf[QB];
#pragma unroll
          for (int i = 0; i < QB; ++i) sf[i] = pack_pair<T>(ds[i][0], ds[i][1]);
#pragma unroll
          for (int db = 0; db < 2 * KS; ++db) {
            const short8 kf = ra_tr_frag(kimg, pb * 32, db, lane);
#pragma unroll
            for (int i = 0; i < QB; ++i) dq[i][db] = Half16<T>::mfma(kf, sf[i], dq[i][db]);
          }
          if (part) {
#pragma unroll
            for (int i = 0; i < QB; ++i) {
              const float4v t = ds[i][0] + ds[i][1];
              e_all[i] += (t[0] + t[1]) + (t[2] + t[3]);
            }
            if (KIND != RA_FARAWAY) {  // tiles of the same offset u = u0 + 16 (kb - i) first add up
              const int u = u0 + 32 * pb;
              if (QB == 2) {
                if (open_u == u - 16) {
                  near(u - 16, open + ds[QB - 1][0]);
                } else {
                  if (open_u != RaDiag::NONE) near(open_u, open);
                  near(u - 16, ds[QB - 1][0]);
                }
                near(u, ds[0][0] + ds[QB - 1][1]);
                open = ds[0][1];
                open_u = u + 16;
              } else {
                near(u, ds[0][0]);
                near(u + 16, ds[0][1]);
              }
            }
          }
        }
      }
      cur = nx;
    }
    if (KIND == RA_FARAWAY) {
      far_lo += below ? ra_sum(e_all) - before : 0.f;
      far_hi += below ? 0.f : ra_sum(e_all) - before;
    }
    return cur;
  };
  while (!cur.done()) cur = sweep(RaKind<RA_PARTIAL>{}, sweep(RaKind<RA_NEAR>{}, sweep(RaKind<RA_FARAWAY>{}, cur)));
  if (SPLIT == 2) {  // the two waves of a row group add up their halves of the keys
    constexpr int F = QB * 8 * KS;
    static_assert((2 * F + 4 * QB) * 64 * (int)sizeof(float) <= 2 * BUF, "the join reuses the images");
    float* x = reinterpret_cast<float*>(smem) + group * F * 64 + lane;
    float* y = reinterpret_cast<float*>(smem) + (2 * F + group * 2 * QB) * 64 + lane;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QB; ++i) y[(half * QB + i) * 64] = e_all[i];
    if (half == 1 && active) {
#pragma unroll
      for (int e = 0; e < F; ++e) x[e * 64] = dq[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3];
    }
    __syncthreads();
    if (half == 0 && active) {
#pragma unroll
      for (int e = 0; e < F; ++e) dq[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3] += x[e * 64];
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) e_all[i] += y[((half ^ 1) * QB + i) * 64];
  }
  if (active && half == 0) {
    T* dqb = ra_base<T>(p.dq, s, packed);
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int q = q0 + 16 * i + lm;
      ra_store<T, KS>(dqb + (int64_t)q * p.dq.row, dq[i], p.scale * drop_lift, g, p.D, q < s.n);
    }
  }
  if (part) {  // the far sums join the ends of their wave's first array; then distances -> buckets
    if (open_u != RaDiag::NONE) near(open_u, open);
    diag.flush();
    if (p.mass) {
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        const int q = q0 + 16 * i + lm;
        const float e = ra_quad_sum(e_all[i]);
        if (half == 0 && g == 0 && q < s.n) {  // once per row; a share of 0 takes nothing, not even NaN
          const float ml = p.mass[bh * p.S + q], mh = p.mass[((int64_t)p.B * p.A + bh) * p.S + q];
          far_lo -= ml != 0.f ? e * ml : 0.f;
          far_hi -= mh != 0.f ? e * mh : 0.f;
        }
      }
    }
    const float lo = wave_sum(far_lo);
    const float hi = wave_sum(far_hi);
    float* const mine = sums + wave * 2 * dlen;
    float* const drops = sums + 2 * RA_WAVES * dlen;
    if (lane == 0) {
      mine[0] += lo;
      mine[2 * bias.far + 62] += hi;
      if (RA_LIFTS<T>) drops[wave] = drop_lift;
    }
    __syncthreads();
    for (int i = tid; i < dlen; i += RA_THREADS) {  // (the eight arrays into the first)
      float t = 0.f;
#pragma unroll
      for (int a = 0; a < 2 * RA_WAVES; ++a) t += sums[a * dlen + i] * (RA_LIFTS<T> ? drops[a >> 1] : 1.0f);
      sums[i] = t;
    }
    __syncthreads();
    ra_bucket_sums<RA_THREADS>(p, sums, bias.far + 31, part, tid);
  }
}

// ------------------------------------------------------------------------------------------------ dK, dV
// One wave = 16 QB keys, sweeps the queries (Q and dO images; SPLIT 2: half of every chunk); the start values of the products and the dropout seeds
// of a chunk's queries in LDS.
template <typename T, int KS, int QB, int SPLIT, bool DROP>
__global__ __launch_bounds__(RA_THREADS) RA_OCC_DKV void rel_attn_dkv_kernel(PdtRelAttn p) {
  constexpr int NH = (KS + 1) / 2, BUF = 2 * NH * RA_IMG + 1024;  // Q | dO | lse, delta, seeds (64 each), 256 spare bytes
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, lm = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RaSpan s = ra_span(p, blockIdx.x);
  constexpr int ROWS = RA_WAVES / SPLIT * 16 * QB;
  const int group = SPLIT == 2 ? wave & 1 : wave, half = SPLIT == 2 ? wave >> 1 : 0;
  const int w0 = blockIdx.y * ROWS, k0 = w0 + group * 16 * QB;
  ra_tail<T>(p, s, p.dk, tid, RA_THREADS);
  ra_tail<T>(p, s, p.dv, tid, RA_THREADS);
  if (w0 >= s.n) return;
  const bool packed = p.cu != nullptr;
  const T* qb_ = ra_base<const T>(p.q, s, packed);
  const T* kb_ = ra_base<const T>(p.k, s, packed);
  const T* vb_ = ra_base<const T>(p.v, s, packed);
  const T* gb_ = ra_base<const T>(p.dout, s, packed);
  const int64_t bh = (int64_t)s.b * p.A + s.h;
  const DropKey dkey = drop_key(p.rng);
  const uint32_t sbh = drop_sample(p.rng, s.b) * p.A + s.h;
  auto stage = [&](int c, int buf) {
    char* m = smem + buf * BUF;
    const int left = s.n - c * RA_CHUNK;
    const uint64_t rows = left >= RA_CHUNK ? ~0ull : (1ull << left) - 1;
    ra_stage<T, NH>(m, qb_ + (int64_t)c * RA_CHUNK * p.q.row, (uint32_t)p.q.row, rows, p.D, lane, wave);
    ra_stage<T, NH>(m + NH * RA_IMG, gb_ + (int64_t)c * RA_CHUNK * p.dout.row, (uint32_t)p.dout.row, rows, p.D, lane, wave);
    // -lse / k2 (wave 0) and -delta (wave 1) of the chunk's queries; waves 2 and 3 read delta again into the spare bytes, so that every
    // wave has the same number of transfers in flight.
    const float* src = p.delta + ((wave == 0 ? (int64_t)p.B * p.A : 0) + bh) * p.S + (int64_t)c * RA_CHUNK;
    const int slot = wave == 0 ? 0 : (wave == 1 ? 1 : 3);
    pdt_lds_dma4(pdt_make_rsrc(src, 256u), m + 2 * NH * RA_IMG + slot * 256, lane < left ? lane * 4u : 0x80000000u);
    if (DROP && tid < 64)
      reinterpret_cast<uint32_t*>(m + 2 * NH * RA_IMG + 512)[tid] = attn_row_seed(dkey, sbh, c * RA_CHUNK + tid);
  };
  auto word = [&](int c) { return s.n - c * RA_CHUNK >= RA_CHUNK ? ~0ull : (1ull << (s.n - c * RA_CHUNK)) - 1; };  // (queries)
  RaChunks cur = ra_chunks(s.n, w0, ROWS, ra_far(p.max_distance), p.table != nullptr);
  cur.next(word);
  short8 kf[QB][KS], vf[QB][KS];
  bool kok[QB];  // (what a lane computes for a key that no query attends to is dropped at the end)
  uint32_t kmul[QB];
  const uint64_t kw = k0 < s.n ? ra_word(p, s, k0 / RA_CHUNK) >> (k0 % RA_CHUNK) : 0;
  const bool active = (kw & (QB == 2 ? 0xFFFFFFFFull : 0xFFFFull)) != 0;  // (a wave's keys lie in one chunk)
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int key = k0 + 16 * i + lm;
    const bool ok = (kw >> (16 * i + lm)) & 1;
    kok[i] = ok;
    kmul[i] = (uint32_t)key * ATT_GOLD;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[i][ks] = ra_gfrag<T>(kb_ + (int64_t)key * p.k.row, ks, p.D, lane, ok);
      vf[i][ks] = ra_gfrag<T>(vb_ + (int64_t)key * p.v.row, ks, p.D, lane, ok);
    }
  }
  stage(cur.c, 0);
  int lift = 0;  // (one for all queries: it goes into P through the bias array)
  if constexpr (RA_LIFTS<T>) {
    const int blocks = (p.S + p.peak_rows - 1) / p.peak_rows, there = (s.n + p.peak_rows - 1) / p.peak_rows * RA_WAVES;
    const uint32_t* const peaks = p.peaks + bh * blocks * RA_WAVES;
    uint32_t top = 0;
    for (int i = lane; i < there; i += 64) top = max(top, peaks[i]);
    lift = ra_lift(ra_wave_max(top), p.drop_scale);
  }
  const float drop_lift = RA_LIFTS<T> ? __uint_as_float((uint32_t)(127 - lift) << 23) : 1.0f;  // 2^-lift
  const RaBias bias = ra_bias_fill<T>(p, reinterpret_cast<float*>(smem + 2 * BUF), s.h, -1, tid, p.max_distance, (float)lift);
  const int boff = ra_bias_lane(bias, lm, g);
  const float k2 = p.scale * LOG2E;
  const uint32_t thr_hi = attn_thr_hi(p.drop_thr);
  float4v dk_[QB][2 * KS], dv_[QB][2 * KS];
#pragma unroll
  for (int i = 0; i < QB; ++i)
#pragma unroll
    for (int db = 0; db < 2 * KS; ++db) { dk_[i][db] = splat4(0.f); dv_[i][db] = splat4(0.f); }
  __syncthreads();  // the bias array is complete
  const float bias_lo = bias.t[0], bias_hi = bias.t[bias.len - 1];
  auto sweep = [&](auto kind, RaChunks cur) {
    constexpr int KIND = decltype(kind)::value;
    while (!cur.done() && cur.kind() == KIND) {
      const int buf = cur.buf;
      RaChunks nx = cur;
      nx.next(word);
      nx.buf ^= 1;
      __syncthreads();  // every wave is done with the other buffer
      if (!nx.done()) {
        stage(nx.c, buf ^ 1);
        if (NH == 1) asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const char* qimg = smem + buf * BUF;
      const char* gimg = qimg + NH * RA_IMG;
      float* const sc_ = reinterpret_cast<float*>(smem + buf * BUF + 2 * NH * RA_IMG);
      // queries that are not there: p = 0 (their start value has arrived as 0)
      if (KIND == RA_PARTIAL && wave == 0 && cur.c * RA_CHUNK + lane >= s.n) sc_[lane] = k2 > 0.f ? -INFINITY : INFINITY;
      __syncthreads();
      if (active) {
        const int u0 = cur.c * RA_CHUNK - k0;  // query - key: the bias array is mirrored
        const float flat = cur.c <= cur.lo ? bias_lo : bias_hi;
#pragma unroll
        for (int pi = 0; pi < 2 / SPLIT; ++pi) {
          const int pb = SPLIT == 2 ? half : pi;
          float4v pp[QB][2], ds[QB][2];
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            const int q16 = pb * 32 + hb * 16;
            const float4v lse = *reinterpret_cast<const float4v*>(sc_ + q16 + 4 * g);
            const float4v del = *reinterpret_cast<const float4v*>(sc_ + 64 + q16 + 4 * g);
            const uint4v sd = *reinterpret_cast<const uint4v*>(sc_ + 128 + q16 + 4 * g);
            float4v sc[QB], dp[QB];
#pragma unroll
            for (int i = 0; i < QB; ++i) { sc[i] = lse; dp[i] = DROP ? splat4(0.f) : del; }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const short8 qf = ra_row_frag(qimg, q16, ks, lane), gf = ra_row_frag(gimg, q16, ks, lane);
#pragma unroll
              for (int i = 0; i < QB; ++i) {
                sc[i] = Half16<T>::mfma(qf, kf[i][ks], sc[i]);
                dp[i] = Half16<T>::mfma(gf, vf[i][ks], dp[i]);
              }
            }
#pragma unroll
            for (int i = 0; i < QB; ++i) {
              float4v t = sc[i] * k2 + (KIND == RA_FARAWAY ? splat4(flat) : ra_bias4(bias, boff, u0 + q16 - 16 * i));
              float4v e = dp[i], pd;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                t[r] = __builtin_amdgcn_exp2f(t[r]);
                const float keep = !DROP ? 1.f : (attn_keep(sd[r], kmul[i], thr_hi) ? p.drop_scale : 0.f);
                pd[r] = DROP ? t[r] * keep : t[r];
                if (DROP) e[r] *= keep;
              }
              pp[i][hb] = pd;
              ds[i][hb] = DROP ? t * (e + del) : t * e;
            }
          }
          short8 pf[QB], sf[QB];
#pragma unroll
          for (int i = 0; i < QB; ++i) { pf[i] = pack_pair<T>(pp[i][0], pp[i][1]); sf[i] = pack_pair<T>(ds[i][0], ds[i][1]); }
#pragma unroll
          for (int db = 0; db < 2 * KS; ++db) {
            const short8 gf = ra_tr_frag(gimg, pb * 32, db, lane), qf = ra_tr_frag(qimg, pb * 32, db, lane);
#pragma unroll
            for (int i = 0; i < QB; ++i) {
              dv_[i][db] = Half16<T>::mfma(gf, pf[i], dv_[i][db]);
              dk_[i][db] = Half16<T>::mfma(qf, sf[i], dk_[i][db]);
            }
          }
        }
      }
      cur = nx;
    }
    return cur;
  };
  while (!cur.done()) cur = sweep(RaKind<RA_PARTIAL>{}, sweep(RaKind<RA_NEAR>{}, sweep(RaKind<RA_FARAWAY>{}, cur)));
  if (SPLIT == 2) {  // the two waves of a key group add up their halves of the queries
    constexpr int F = QB * 8 * KS;
    static_assert(4 * F * 64 * (int)sizeof(float) <= 2 * BUF, "the join reuses the images");
    float* x = reinterpret_cast<float*>(smem) + group * 2 * F * 64 + lane;
    __syncthreads();
    if (half == 1 && active) {
#pragma unroll
      for (int e = 0; e < F; ++e) {
        x[e * 64] = dk_[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3];
        x[(F + e) * 64] = dv_[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3];
      }
    }
    __syncthreads();
    if (half == 1) return;
    if (active) {
#pragma unroll
      for (int e = 0; e < F; ++e) {
        dk_[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3] += x[e * 64];
        dv_[e / (8 * KS)][(e / 4) % (2 * KS)][e & 3] += x[(F + e) * 64];
      }
    }
  }
  T* dkb = ra_base<T>(p.dk, s, packed);
  T* dvb = ra_base<T>(p.dv, s, packed);
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int key = k0 + 16 * i + lm;
    if (!kok[i]) {
#pragma unroll
      for (int db = 0; db < 2 * KS; ++db) dk_[i][db] = dv_[i][db] = splat4(0.f);
    }
    ra_store<T, KS>(dkb + (int64_t)key * p.dk.row, dk_[i], p.scale * drop_lift, g, p.D, key < s.n);
    ra_store<T, KS>(dvb + (int64_t)key * p.dv.row, dv_[i], drop_lift, g, p.D, key < s.n);
  }
}

// ------------------------------------------------------------------------------------------------ backward, S <= 16 W
// One workgroup of W waves owns a whole (batch, head): every input is read once and every probability computed once.
// First each wave takes 16 query rows against all keys, with p and dp of the whole row in registers: delta = sum of p dp is
// formed from them (neither the output nor its rounding enters), ds follows, and dQ.  Then P and dS go to LDS as 16-bit
// images in the place of K and V, and each wave takes 16 keys: their columns of P and dS, read transposed, are the operands
// of dV and dK against the images of dO and Q.  With 64 columns and 128 rows the place holds 64 keys' worth, so this runs in
// two passes, two waves sharing the columns of 16 keys; otherwise in one.
// Bound by memory at the training shapes: 7 row reads and writes of 16-bit values per element instead of the two sweeps' 11.
template <typename T, int KS, int W, bool DROP>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(KS <= 2 ? 4 : 2, 8))) void rel_attn_bwd_short_kernel(PdtRelAttn p) {
  constexpr int NH = (KS + 1) / 2, R = 16 * W, NC = R / RA_CHUNK;  // NC 64-row chunks; an image is [NC][NH] chunk images
  constexpr int IMG = NC * NH * RA_IMG;
  constexpr int PASSES = NC > NH ? 2 : 1, SPLIT = PASSES;          // key passes; waves that share 16 keys
  constexpr int CK = NC / PASSES;                                  // 64-key chunks of a pass
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* const qimg = smem;
  char* const gimg = smem + IMG;
  char* const kimg = smem + 2 * IMG;  // K | V, later P | dS
  char* const vimg = smem + 3 * IMG;
  const int tid = threadIdx.x, lane = tid & 63, lm = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RaSpan s = ra_span(p, blockIdx.x);
  float* part = p.dtable_part ? p.dtable_part + (int64_t)s.b * p.buckets * p.A + s.h : nullptr;
  ra_tail<T>(p, s, p.dq, tid, 64 * W);
  ra_tail<T>(p, s, p.dk, tid, 64 * W);
  ra_tail<T>(p, s, p.dv, tid, 64 * W);
  if (s.n == 0) {
    if (part)
      for (int i = tid; i < p.buckets; i += 64 * W) part[(int64_t)i * p.A] = 0.f;
    return;
  }
  const bool packed = p.cu != nullptr;
  uint64_t rows[NC], keys[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int left = s.n - c * RA_CHUNK;
    rows[c] = left <= 0 ? 0 : (left >= RA_CHUNK ? ~0ull : (1ull << left) - 1);
    keys[c] = ra_word(p, s, c);
  }
  auto stage = [&](char* img, const PdtRelView& v, const uint64_t (&on)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      ra_stage<T, NH, W>(img + c * NH * RA_IMG, ra_base<const T>(v, s, packed) + (int64_t)c * RA_CHUNK * v.row, (uint32_t)v.row, on[c], p.D, lane, wave);
  };
  stage(kimg, p.k, keys);
  stage(vimg, p.v, keys);
  stage(qimg, p.q, rows);
  stage(gimg, p.dout, rows);
  const int q = 16 * wave + lm;
  const RaBias bias = ra_bias_fill<T, 64 * W>(p, reinterpret_cast<float*>(smem + 4 * IMG), s.h, 1, tid, min(p.max_distance, 128));
  const float k2 = p.scale * LOG2E;
  // what the products start from, so that scores come out with lse subtracted (rows that are not there: p = 0)
  float nlse = (q < s.n ? -p.lse[((int64_t)s.b * p.A + s.h) * p.S + q] : -INFINITY) / k2;
  const int boff = ra_bias_lane(bias, lm, g);
  const uint32_t seed = DROP ? attn_row_seed(drop_key(p.rng), drop_sample(p.rng, s.b) * p.A + s.h, q) : 0u;
  const uint32_t thr_hi = attn_thr_hi(p.drop_thr), kmul0 = (uint32_t)(4 * g) * ATT_GOLD;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  uint32_t* const tops = reinterpret_cast<uint32_t*>(bias.t + 4 * bias.len);
  if constexpr (RA_LIFTS<T>) {  // the largest |dout|, over what this wave has staged
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NC * NH; ++i)
#pragma unroll
      for (int u = 0; u < 8 / W; ++u) top = ra_top(top, *reinterpret_cast<const short8*>(gimg + i * RA_IMG + (u * W + wave) * 1024 + lane * 16));
    top = ra_wave_max(top);
    if (lane == 0) tops[wave] = top;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  int lift = 0;
  if constexpr (RA_LIFTS<T>) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, tops[i]);
    lift = __builtin_amdgcn_readfirstlane(ra_lift(top, p.drop_scale));
    nlse += lift / k2;
  }
  const float drop_lift = RA_LIFTS<T> ? __uint_as_float((uint32_t)(127 - lift) << 23) : 1.0f;  // 2^-lift

  // ---- rows: p, dp, delta, ds, dQ.  (Waves up to the end of the last 32 rows take part: their rows are zero.)
  const bool active = 16 * wave < ((s.n + 31) & ~31);
  float4v ds[W];
  short8 pp[W / 2], sf[W / 2];
#pragma unroll
  for (int pb = 0; pb < W / 2; ++pb) pp[pb] = sf[pb] = short8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int kb = 0; kb < W; ++kb) ds[kb] = splat4(0.f);
  if (active) {
    short8 qf[KS], df[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = ra_row_frag(qimg + (wave >> 2) * NH * RA_IMG, 16 * (wave & 3), ks, lane);
      df[ks] = ra_row_frag(gimg + (wave >> 2) * NH * RA_IMG, 16 * (wave & 3), ks, lane);
    }
    float4v dp[W], d4 = splat4(0.f);
#pragma unroll
    for (int pb = 0; pb < W / 2; ++pb) {
      float4v pd[2];
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        const int kb = 2 * pb + hb;
        const uint32_t tile = (uint32_t)(keys[kb >> 2] >> ((kb & 3) * 16)) & 0xFFFFu;  // (wave-uniform)
        dp[kb] = pd[hb] = splat4(0.f);
        if (!tile) continue;
        float4v sc = splat4(nlse), e = splat4(0.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          sc = Half16<T>::mfma(ra_row_frag(kimg + (kb >> 2) * NH * RA_IMG, (kb & 3) * 16, ks, lane), qf[ks], sc);
          e = Half16<T>::mfma(ra_row_frag(vimg + (kb >> 2) * NH * RA_IMG, (kb & 3) * 16, ks, lane), df[ks], e);
        }
        float4v t = sc * k2 + ra_bias4(bias, boff, 16 * (kb - wave));
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = __builtin_amdgcn_exp2f(t[r]);
        // (selected in every tile: a branch between a product and its use has cost the wait in front of that use, see
        // tools/mfma_hazards.py)
        const uint32_t bits = tile >> (4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = (bits >> r) & 1 ? t[r] : 0.f;
        ds[kb] = pd[hb] = t;
        if (DROP) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float keep = attn_keep(seed, kmul0 + (uint32_t)(kb * 16 + r) * ATT_GOLD, thr_hi) ? p.drop_scale : 0.f;
            pd[hb][r] *= keep;
            e[r] *= keep;
          }
        }
        d4 += t * e;
        dp[kb] = e;
      }
      pp[pb] = pack_pair<T>(pd[0], pd[1]);
    }
    const float delta = ra_quad_sum((d4[0] + d4[1]) + (d4[2] + d4[3])) * drop_lift;  // (d4: with the lift of p)
    float4v dq[2 * KS];
#pragma unroll
    for (int db = 0; db < 2 * KS; ++db) dq[db] = splat4(0.f);
#pragma unroll
    for (int pb = 0; pb < W / 2; ++pb) {
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) ds[2 * pb + hb] *= dp[2 * pb + hb] - delta;
      sf[pb] = pack_pair<T>(ds[2 * pb], ds[2 * pb + 1]);
      if (((keys[pb >> 1] >> ((pb & 1) * 32)) & 0xFFFFFFFFull) == 0) continue;
#pragma unroll
      for (int db = 0; db < 2 * KS; ++db)
        dq[db] = Half16<T>::mfma(ra_tr_frag(kimg + (pb >> 1) * NH * RA_IMG, (pb & 1) * 32, db, lane), sf[pb], dq[db]);
    }
    ra_store<T, KS>(ra_base<T>(p.dq, s, packed) + (int64_t)q * p.dq.row, dq, p.scale * drop_lift, g, p.D, q < s.n);
  }

  // ---- keys: dV and dK.  A pass: P and dS of its keys as [query][64 keys] images, then 16 keys per wave.
  T* dkb = ra_base<T>(p.dk, s, packed);
  T* dvb = ra_base<T>(p.dv, s, packed);
  const int nqb = (s.n + 31) >> 5;
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass) {
    const int kblk = pass * 4 * CK + (SPLIT == 2 ? wave & 3 : wave), part_d = SPLIT == 2 ? wave >> 2 : 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (this wave is done with the place)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kb = 0; kb < 4 * CK; ++kb) {  // this wave's 16 queries x 4 CK key blocks: four keys (8 bytes) per lane and block
      const int at = pass * 4 * CK + kb, pos = q & (RA_CHUNK - 1);
      const int off = ((q >> 6) * CK + (kb >> 2)) * RA_IMG + pos * 128 + (((2 * (kb & 3) + (g >> 1)) ^ (pos & 6)) << 4) + (g & 1) * 8;
      const int4v a = __builtin_bit_cast(int4v, pp[at >> 1]), c = __builtin_bit_cast(int4v, sf[at >> 1]);
      *reinterpret_cast<int2v*>(kimg + off) = at & 1 ? int2v{a[2], a[3]} : int2v{a[0], a[1]};
      *reinterpret_cast<int2v*>(vimg + off) = at & 1 ? int2v{c[2], c[3]} : int2v{c[0], c[1]};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const int key = 16 * kblk + lm;
    constexpr int DB = 2 * KS / SPLIT > 0 ? 2 * KS / SPLIT : 1;  // 16-column blocks of this wave
    float4v dk_[DB], dv_[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) { dk_[i] = splat4(0.f); dv_[i] = splat4(0.f); }
    if (((keys[kblk >> 2] >> ((kblk & 3) * 16)) & 0xFFFFu) != 0) {
      const int kin = kblk - pass * 4 * CK;  // block within the pass
      for (int qb = 0; qb < nqb; ++qb) {
        const int base = (qb >> 1), r0 = (qb & 1) * 32;
        const short8 pf = ra_tr_frag(kimg + (base * CK + (kin >> 2)) * RA_IMG, r0, kin & 3, lane);
        const short8 tf = ra_tr_frag(vimg + (base * CK + (kin >> 2)) * RA_IMG, r0, kin & 3, lane);
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const int db = part_d * DB + i;
          dv_[i] = Half16<T>::mfma(ra_tr_frag(gimg + base * NH * RA_IMG, r0, db, lane), pf, dv_[i]);
          dk_[i] = Half16<T>::mfma(ra_tr_frag(qimg + base * NH * RA_IMG, r0, db, lane), tf, dk_[i]);
        }
      }
    }
    if constexpr (DB % 2 == 0) {
      const int c0 = part_d * DB * 16;
      ra_store<T, DB / 2>(dkb + (int64_t)key * p.dk.row + c0, dk_, p.scale * drop_lift, g, p.D - c0, key < s.n);
      ra_store<T, DB / 2>(dvb + (int64_t)key * p.dv.row + c0, dv_, drop_lift, g, p.D - c0, key < s.n);
    } else {  // one block: four columns (8 bytes) per lane
      const int col = part_d * 16 + 4 * g;
      if (key < s.n && col < p.D) {
        const float4v a = dk_[0] * (p.scale * drop_lift), c = dv_[0] * drop_lift;
        *reinterpret_cast<int2v*>(dkb + (int64_t)key * p.dk.row + col) = int2v{cvt_pk<T>(a[0], a[1]), cvt_pk<T>(a[2], a[3])};
        *reinterpret_cast<int2v*>(dvb + (int64_t)key * p.dv.row + col) = int2v{cvt_pk<T>(c[0], c[1]), cvt_pk<T>(c[2], c[3])};
      }
    }
  }

  // ---- table gradient: the diagonals of this wave's rows (a tile per offset 16 (kb - wave): each entry is written once,
  // the part W of a tile that belongs to the next offset is carried), then distances -> buckets
  if (!part) return;
  constexpr int TOP = R - 1, DLEN = 2 * R + 16;
  float* const sums = reinterpret_cast<float*>(smem);
  __syncthreads();
  for (int i = tid; i < 4 * W * DLEN; i += 64 * W) sums[i] = 0.f;
  __syncthreads();
  {
    float* d = sums + (wave * 4 + g) * DLEN + TOP - 16 * wave + 4 * g - lm;
    float carry = 0.f;
#pragma unroll
    for (int kb = 0; kb < W; ++kb) {
      const float4v t = ds[kb];
      const float n = ra_diag_n(t), w = ra_diag_w(t);
      d[16 * kb] = n + carry;
      carry = w;
    }
    if (lm >= 13) d[16 * W] = carry;
  }
  __syncthreads();
  for (int i = tid; i < DLEN; i += 64 * W) {
    float t = 0.f;
#pragma unroll 8
    for (int a = 0; a < 4 * W; ++a) t += sums[a * DLEN + i];
    sums[i] = t * drop_lift;
  }
  __syncthreads();
  ra_bucket_sums<64 * W>(p, sums, TOP, part, tid);
}

// ------------------------------------------------------------------------------------------------ helpers
// key mask [B][S] (1 or 4 bytes per key, non-zero = attended) -> one bit per key; one wave per 64 keys
__global__ __launch_bounds__(256) void rel_attn_mask_kernel(const void* mask, int bytes, int64_t stride, int S, int words,
                                                            int total, uint64_t* bits) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= total) return;
  const int b = i / words, c = i - b * words, k = c * 64 + lane;
  bool on = false;
  if (k < S) {
    const int64_t at = (int64_t)b * stride + k;
    on = bytes == 1 ? ((const uint8_t*)mask)[at] != 0 : ((const int32_t*)mask)[at] != 0;
  }
  const uint64_t w = __ballot(on);
  if (lane == 0) bits[i] = w;
}

// more dynamic LDS than 64 KiB needs the attribute; set once per kernel and device (not a stream operation: done at the
// first launch, i.e. in the warm-up of a step that is captured later)
static int ra_allow_lds(const void* kern, size_t bytes) {
  static std::mutex mu;
  static std::unordered_set<const void*> done[64];
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return (int)e;
  std::lock_guard<std::mutex> lock(mu);
  if (bytes > 160 * 1024 || dev < 0 || dev >= 64) return -3;
  if (done[dev].count(kern)) return 0;
  const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e != hipSuccess) return (int)e;
  done[dev].insert(kern);
  return 0;
}

// Shape of a workgroup.  A wave takes two 16-row blocks, so that both use every row it reads from LDS.  128 rows: four waves
// with 32 rows each.  64 rows: two pairs of waves, a pair shares 32 rows and splits every chunk - up to half as slow again per
// row in long sequences (2 x 4096 tokens, 16 heads: forward 231 against 189 us), but sequences of up to 64 rows keep all waves
// busy, and small batches reach more CUs (12 heads, 1 x 300 tokens: backward 29.5 against 35.0 us, 1 x 2000: 100 against
// 119 us).  Compared by rounds over the `slots` workgroups that run at a time: those of the default max_distance of 128.  The
// arrays of dQ take 96 bytes more per unit of distance; at 512 one of its workgroups fills a CU (32 x 512 tokens, 12 heads: 183
// instead of 78 us; forward and dK / dV stay), which this rule does not weigh.
enum { RA_FWD, RA_DQ, RA_DKV, RA_SHORT };
static int ra_rows(const PdtRelAttn& p, int which) {
  const int64_t len = p.cu ? (p.B ? p.T / p.B : 0) : p.S;  // (packed: the average)
  if (len <= 64) return 64;
  const int64_t slots = 256 * (which == RA_DKV || p.D > 64 ? 2 : 3), heads = (int64_t)p.B * p.A;
  const int64_t full = (heads * ((len + 127) / 128) + slots - 1) / slots, half = (heads * ((len + 63) / 64) + slots - 1) / slots;
  return half * 4 < full * 5 ? 64 : 128;
}

static size_t ra_bias_bytes(const PdtRelAttn& p) { return (size_t)4 * ra_bias_len(p.max_distance) * sizeof(float); }

// (a launch counts its threads along x in 32 bits)
static bool ra_too_many(const PdtRelAttn& p, int threads) { return (int64_t)p.B * p.A * threads > 0xFFFFFFFFll; }

template <typename KernT>
static int ra_launch(KernT kern, const PdtRelAttn& p, int rows_per_block, size_t lds, hipStream_t stream) {
  if (ra_too_many(p, RA_THREADS)) return -3;
  if (int e = ra_allow_lds((const void*)kern, lds)) return e;
  hipLaunchKernelGGL(kern, dim3(p.B * p.A, (p.S + rows_per_block - 1) / rows_per_block), dim3(RA_THREADS), lds, stream, p);
  return (int)hipGetLastError();
}

// sequences that one workgroup of the short backward kernel holds: 64 rows in four waves, 128 in eight
static int ra_short_rows(const PdtRelAttn& p) { return p.S <= 64 ? 64 : (p.S <= 128 ? 128 : 0); }
template <typename T, int KS, int W, bool DROP>
static int ra_launch_short(const PdtRelAttn& p, hipStream_t st) {
  constexpr int NH = (KS + 1) / 2, R = 16 * W;
  const size_t work = (size_t)4 * (R / RA_CHUNK) * NH * RA_IMG;
  static_assert((size_t)4 * W * (2 * R + 16) * sizeof(float) <= (size_t)4 * (R / RA_CHUNK) * NH * RA_IMG, "diagonal sums reuse the images");
  const size_t lds = work + (size_t)4 * ra_bias_len(p.max_distance < 128 ? p.max_distance : 128) * sizeof(float) + W * sizeof(uint32_t);
  auto kern = rel_attn_bwd_short_kernel<T, KS, W, DROP>;
  if (ra_too_many(p, 64 * W)) return -3;
  if (int e = ra_allow_lds((const void*)kern, lds)) return e;
  hipLaunchKernelGGL(kern, dim3(p.B * p.A), dim3(64 * W), lds, st, p);
  return (int)hipGetLastError();
}

template <typename T, int KS, bool DROP>
static int ra_dispatch(int which, const PdtRelAttn& p, hipStream_t st) {
  constexpr int NH = (KS + 1) / 2;
  if (which == RA_SHORT) return ra_short_rows(p) == 64 ? ra_launch_short<T, KS, 4, DROP>(p, st) : ra_launch_short<T, KS, 8, DROP>(p, st);
  const int rows = ra_rows(p, which);
  const size_t imgs = (size_t)4 * NH * RA_IMG, tab = ra_bias_bytes(p);
  if (which == RA_FWD) {
    const size_t zones = p.mass ? (size_t)2 * RA_WAVES * 32 * sizeof(float) : 0;
    return rows == 128 ? ra_launch(rel_attn_fwd_kernel<T, KS, 2, 1, DROP>, p, rows, imgs + 512 + tab + zones, st)
                       : ra_launch(rel_attn_fwd_kernel<T, KS, 2, 2, DROP>, p, rows, imgs + 512 + tab + zones, st);
  }
  if (which == RA_DQ) {
    const size_t diag = p.dtable_part ? (size_t)RA_WAVES * (2 * ra_diag_len(p.max_distance) + 1) * sizeof(float) : 0;
    return rows == 128 ? ra_launch(rel_attn_dq_kernel<T, KS, 2, 1, DROP>, p, rows, imgs + 512 + tab + diag, st)
                       : ra_launch(rel_attn_dq_kernel<T, KS, 2, 2, DROP>, p, rows, imgs + 512 + tab + diag, st);
  }
  // (beyond 64 columns the accumulators of two blocks of dK and dV do not fit the registers: one block per wave)
  if constexpr (KS > 2) return ra_launch(rel_attn_dkv_kernel<T, KS, 1, 1, DROP>, p, 64, imgs + 2048 + tab, st);
  else
    return rows == 128 ? ra_launch(rel_attn_dkv_kernel<T, KS, 2, 1, DROP>, p, rows, imgs + 2048 + tab, st)
                       : ra_launch(rel_attn_dkv_kernel<T, KS, 2, 2, DROP>, p, rows, imgs + 2048 + tab, st);
}
template <typename T>
static int ra_dispatch_ks(int which, const PdtRelAttn& p, hipStream_t st) {
  const bool drop = p.drop_thr != 0;
  switch ((p.D + 31) / 32) {
    case 1: return drop ? ra_dispatch<T, 1, true>(which, p, st) : ra_dispatch<T, 1, false>(which, p, st);
    case 2: return drop ? ra_dispatch<T, 2, true>(which, p, st) : ra_dispatch<T, 2, false>(which, p, st);
    case 3: return drop ? ra_dispatch<T, 3, true>(which, p, st) : ra_dispatch<T, 3, false>(which, p, st);
    case 4: return drop ? ra_dispatch<T, 4, true>(which, p, st) : ra_dispatch<T, 4, false>(which, p, st);
  }
  return -3;
}
static int ra_run(int dtype, int which, const PdtRelAttn& p, hipStream_t st) {
  return dtype == PDT_F16 ? ra_dispatch_ks<_Float16>(which, p, st) : ra_dispatch_ks<__bf16>(which, p, st);
}

static int ra_check(int dtype, const PdtRelAttn& p) {
  if (dtype != PDT_F16 && dtype != PDT_BF16) return -1;
  if (p.B < 0 || p.S < 0 || p.A <= 0 || p.D <= 0 || p.D > 128 || p.D % 8) return -3;
  if ((int64_t)p.B * p.A > 0x7FFFFFFF || (p.S + RA_CHUNK - 1) / RA_CHUNK > 65535) return -3;
  const PdtRelView* views[] = {&p.q, &p.k, &p.v, &p.o, &p.o_lo, &p.dout, &p.dq, &p.dk, &p.dv, nullptr};
  for (int i = 0; views[i]; ++i)  // 16-byte rows, and 64 rows within the 31-bit window of a transfer
    if (views[i]->p && (views[i]->row % 8 || views[i]->head % 8 || views[i]->batch % 8 || views[i]->row < 0 ||
                        views[i]->row > (1 << 23) || (uintptr_t)views[i]->p % 16))
      return -4;
  if (!p.q.p || !p.k.p || !p.v.p || !p.o.p) return -2;
  if (p.mask && ((p.mask_bytes != 1 && p.mask_bytes != 4) || p.mask_bits)) return -2;
  if (p.table && (p.buckets < 4 || p.buckets % 2 || p.buckets > 4 * RA_MAX_STEPS || p.max_distance <= p.buckets / 4 ||
                  p.max_distance > RA_MAX_FAR))
    return -5;
  if (!p.table && p.max_distance != 0) return -5;
  return 0;
}

}  // namespace pdt

using namespace pdt;

extern "C" int pdt_rel_attn_mask(const void* mask, int bytes, int64_t stride, int B, int S, uint64_t* bits, void* stream) {
  if (!mask || !bits || (bytes != 1 && bytes != 4) || B < 0 || S < 0) return -1;
  const int words = (S + 63) / 64;
  const int64_t total = (int64_t)B * words;
  if (total == 0) return 0;
  if (total > 0x7FFFFFFF) return -3;
  hipLaunchKernelGGL(rel_attn_mask_kernel, dim3((unsigned)((total + 3) / 4)), dim3(256), 0, (hipStream_t)stream, mask, bytes,
                     stride, S, words, (int)total, bits);
  return (int)hipGetLastError();
}

extern "C" int pdt_rel_attn_fwd(int dtype, const PdtRelAttn* a, void* stream) {
  if (int e = ra_check(dtype, *a)) return e;
  hipStream_t st = (hipStream_t)stream;
  if (a->B == 0 || a->S == 0) return 0;
  return ra_run(dtype, RA_FWD, *a, st);
}

extern "C" int pdt_rel_attn_uses_low(int S) { return S > 128 ? 1 : 0; }

extern "C" int pdt_rel_attn_dtable_rows(const PdtRelAttn* a) {
  if (ra_short_rows(*a)) return a->B;
  const int rows = ra_rows(*a, RA_DQ);
  return a->B * ((a->S + rows - 1) / rows);
}

extern "C" int64_t pdt_rel_attn_peaks(int dtype, const PdtRelAttn* a) {  // one entry per wave of dQ
  if (dtype != PDT_F16 || ra_short_rows(*a)) return 0;
  const int rows = ra_rows(*a, RA_DQ);
  return (int64_t)a->B * a->A * ((a->S + rows - 1) / rows) * RA_WAVES;
}

extern "C" int pdt_rel_attn_bwd(int dtype, const PdtRelAttn* a, void* stream) {
  if (int e = ra_check(dtype, *a)) return e;
  if (!a->dout.p || !a->dq.p || !a->dk.p || !a->dv.p) return -2;
  if (a->B > 0 && a->S > 0 && (!a->lse || !a->delta)) return -2;
  if (a->dtable_part && !a->table) return -2;
  hipStream_t st = (hipStream_t)stream;
  if (a->B == 0 || a->S == 0) return 0;
  if (ra_short_rows(*a)) return ra_run(dtype, RA_SHORT, *a, st);
  if (pdt_rel_attn_peaks(dtype, a) && !a->peaks) return -2;
  PdtRelAttn p = *a;
  p.peak_rows = ra_rows(p, RA_DQ);
  if (int e = ra_run(dtype, RA_DQ, p, st)) return e;
  return ra_run(dtype, RA_DKV, p, st);
}
