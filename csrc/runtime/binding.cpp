// Torch-facing runtime of the gfx950 kernel library: tensor checks, stream plumbing, and the fused
// encoder-layer forward/backward that chains the kernels (the per-layer "schedule" lives here in C++,
// so one Python call issues all launches of a layer on the current HIP stream).
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/hip/HIPEvent.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <memory>
#include <functional>
#include <mutex>
#include <unordered_map>
#include <vector>

#include "../kernels/api.h"

namespace py = pybind11;
using at::Tensor;

namespace {

// PyTorch-ROCm names its device type "cuda"; these are the guard / stream classes that accept it.
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
void* cur_stream() { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

// Weight-gradient lane: in the layer backward the wgrad GEMM of a projection does not feed anything later in the
// layer, so it can be issued on a second HIP stream and run concurrently with the dgrad chain.  Measured on
// MI355X (BERT-large, seq 128): +5 % step throughput at 8192 tokens per micro-batch and +1.6 % at 4096 (the
// GEMMs of such a micro-batch leave CUs idle in their tail rounds, the concurrent kernel fills them), but
// -1.3 % at 16384 and -3.4 % at 32768 tokens, where every GEMM fills the chip by itself and two of them only
// compete for L2.  Mode 1 (default) therefore uses the lane up to 12288 tokens; PDT_WGRAD_STREAM=0 never, =2
// always.  Fork = event on the main stream the side stream
// waits for; join = event on the side stream the main stream waits for before the layer returns, which also
// makes the caching allocator's stream-ordered reuse of this layer's temporaries safe.
using Stream = c10::hip::HIPStreamMasqueradingAsCUDA;
using StreamGuard = c10::hip::HIPStreamGuardMasqueradingAsCUDA;
int g_wgrad_mode = [] {
  const char* e = std::getenv("PDT_WGRAD_STREAM");
  return (e && e[0] >= '0' && e[0] <= '2') ? e[0] - '0' : 1;
}();
constexpr int kWgradLaneMaxTokens = 12288;
// Deferred mode (set_wgrad_defer(true), used by Engine.accumulate for every backward of an accumulation window but
// the last): short micro-batches are bound by how fast the host can enqueue, and the four forks and the join of a
// layer are 10 of its ~25 runtime calls.  A deferred lane queues the layer's weight-gradient GEMMs, issues them
// behind ONE fork at the end of the layer and does not join: nothing on the main stream reads those gradients
// before the backward pass is over.  The tensors the queued GEMMs read are kept alive (per main stream) until
// wgrad_join() has made the main stream wait for the side stream, which the caller does once, after backward().
bool g_wgrad_defer = false;
std::mutex g_defer_mu;
std::unordered_map<int64_t, std::vector<Tensor>> g_defer_held;  // by main-stream id
class WgradLane {
 public:
  explicit WgradLane(bool enabled, bool defer = false)
      : on_(enabled), defer_(enabled && defer), main_(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA()), side_(main_) {
    if (on_) side_ = side_stream(main_.device_index());
  }
  // run `fn` (kernel launches + its temporaries) on the side stream, after everything issued so far on main
  // (deferred: after everything issued on main up to finish()); `reads` are the tensors it reads
  template <typename F>
  void run(F&& fn, std::initializer_list<Tensor> reads = {}) {
    if (!on_) { fn(); return; }
    if (defer_) {
      pending_.emplace_back(std::forward<F>(fn));
      keep_.insert(keep_.end(), reads.begin(), reads.end());
      return;
    }
    event(next_++).record(main_);
    event(next_ - 1).block(side_);
    StreamGuard g(side_);
    fn();
    used_ = true;
  }
  // end of the layer: join (or, deferred, fork once and issue what was queued)
  void finish() {
    if (defer_ && !pending_.empty()) {
      event(next_++).record(main_);
      event(next_ - 1).block(side_);
      {
        StreamGuard g(side_);
        for (auto& fn : pending_) fn();
      }
      pending_.clear();
      std::lock_guard<std::mutex> lock(g_defer_mu);
      auto& held = g_defer_held[(int64_t)main_.id()];
      held.insert(held.end(), keep_.begin(), keep_.end());
      keep_.clear();
      return;
    }
    join();
  }
  void join() {
    if (!on_ || !used_) return;
    event(next_++).record(side_);
    event(next_ - 1).block(main_);
    used_ = false;
  }
  // (queued launches are only ever issued by finish(): they capture the caller's locals, which are gone by the time
  // a destructor runs during stack unwinding)
  ~WgradLane() { pending_.clear(); join(); }
  // make the current stream wait for the side stream and drop the tensors kept for it (see g_wgrad_defer)
  static void join_deferred() {
    Stream main = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA();
    std::vector<Tensor> drop;
    {
      std::lock_guard<std::mutex> lock(g_defer_mu);
      auto it = g_defer_held.find((int64_t)main.id());
      if (it == g_defer_held.end() || it->second.empty()) return;
      drop.swap(it->second);
    }
    Stream side = side_stream(main.device_index());
    at::cuda::CUDAEvent& e = event(15);
    e.record(side);
    e.block(main);
    // (`drop` is released here: the caching allocator hands the blocks back to the stream they belong to, whose
    // later work is ordered behind the wait above)
  }

 private:
  static Stream side_stream(c10::DeviceIndex dev) {
    static std::vector<std::unique_ptr<Stream>> streams(64);
    if (!streams[dev]) streams[dev] = std::make_unique<Stream>(c10::hip::getStreamFromPoolMasqueradingAsCUDA(false, dev));
    return *streams[dev];
  }
  // events are re-recorded every layer: a small per-thread ring, never destroyed while work may reference them
  static at::cuda::CUDAEvent& event(int i) {
    static thread_local std::vector<std::unique_ptr<at::cuda::CUDAEvent>> ring(16);
    auto& e = ring[i & 15];
    if (!e) e = std::make_unique<at::cuda::CUDAEvent>();
    return *e;
  }
  bool on_, defer_, used_ = false;
  int next_ = 0;
  Stream main_, side_;
  std::vector<std::function<void()>> pending_;
  std::vector<Tensor> keep_;
};

int dt_code(const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return PDT_F16;
  if (t.scalar_type() == at::kBFloat16) return PDT_BF16;
  TORCH_CHECK(false, "expected a float16/bfloat16 tensor, got ", t.scalar_type());
}
// Serialized debug mode (PDT_DEBUG_SYNC=1 or set_debug_sync(true)): the device is drained after every native
// launch, so an asynchronous fault or a sticky error is reported at the op that caused it instead of at the
// next unrelated synchronisation point.  Kernels of different streams never overlap in this mode, which also
// makes it the A/B switch for a suspected stream-ordering bug (a failure that disappears here is an ordering bug).
bool g_debug_sync = [] {
  const char* e = std::getenv("PDT_DEBUG_SYNC");
  return e && e[0] == '1';
}();
int64_t g_debug_sync_count = 0;
void check(int err, const char* what) {
  TORCH_CHECK(err == 0, "pdt kernel launch failed in ", what, ": code ", err,
              err < 0 ? " (argument check)" : " (hipError_t)");
  if (g_debug_sync) {
    const hipError_t e = hipDeviceSynchronize();
    ++g_debug_sync_count;
    TORCH_CHECK(e == hipSuccess, "pdt kernel faulted in ", what, ": ", hipGetErrorString(e));
  }
}
void chk16(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be 16-bit float");
  TORCH_CHECK(t.stride(-1) == 1, name, " must have unit inner stride");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " must be 16-byte aligned");
}
void chkf32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous(), name,
              " must be a contiguous fp32 GPU tensor");
}
uint32_t thr16(double p) { return p <= 0.0 ? 0u : (uint32_t)std::lround(p * 65536.0); }
float keep_scale(double p) { return p <= 0.0 ? 1.0f : (float)(1.0 / (1.0 - p)); }

using OptTensor = c10::optional<Tensor>;
// `sids` (optional int32 [B] on the GPU): global sample ids - the dropout counters of row r of a [B*seq, H]
// activation then derive from (sids[r / seq], r % seq), see PdtRng in api.h.
// `rowmap` (optional int32 [T] on the GPU): unpadded activations - the dropout row of every packed row (PdtRng::row_table).
PdtRng make_rng(const Tensor& state, int64_t micro, int64_t site, const OptTensor& sids = c10::nullopt, int64_t seq = 1,
                int64_t batch = -1, const OptTensor& rowmap = c10::nullopt) {
  TORCH_CHECK(state.is_cuda() && state.scalar_type() == at::kLong && state.numel() >= 2, "rng state: int64[2] on GPU");
  PdtRng r{reinterpret_cast<const uint64_t*>(state.data_ptr<int64_t>()), (uint32_t)micro, (uint32_t)site, nullptr, 1u, 0u};
  if (sids.has_value()) {
    TORCH_CHECK(sids->is_cuda() && sids->scalar_type() == at::kInt && sids->is_contiguous() && sids->dim() == 1,
                "sample_ids must be a contiguous int32 [B] GPU tensor");
    // (a sample has the 512 rows from id * 512 on: ids of longer samples come in steps of several, NativeRuntime.sample_blocks)
    TORCH_CHECK(seq >= 1, "sample-keyed dropout: at least one token per sample");
    TORCH_CHECK(batch < 0 || sids->numel() == batch, "sample_ids has ", sids->numel(), " entries for a batch of ", batch);
    TORCH_CHECK(sids->numel() * seq < std::min(int64_t(1) << 23, (int64_t(1) << 32) / seq),
                "sample-keyed dropout: too many rows for the exact row / seq trick");
    r.sample_ids = sids->data_ptr<int32_t>();
    r.seq = (uint32_t)seq;
    r.seq_magic = seq == 1 ? 0u : (uint32_t)(((uint64_t(1) << 32) + (uint64_t)seq - 1) / (uint64_t)seq);
  }
  if (rowmap.has_value()) {
    TORCH_CHECK(rowmap->is_cuda() && rowmap->scalar_type() == at::kInt && rowmap->is_contiguous() && rowmap->dim() == 1,
                "rowmap must be a contiguous int32 [T] GPU tensor");
    r.row_table = reinterpret_cast<const uint32_t*>(rowmap->data_ptr<int32_t>());
  }
  return r;
}

// ---------------------------------------------------------------------------------------------------
// GEMM wrappers.  2-D operands; leading dimension = stride(0).
// ---------------------------------------------------------------------------------------------------
// Column-sum finishing jobs (bias / gamma / beta gradients) of one layer backward, launched together at its end: with
// short micro-batches a layer's backward is a chain of ~15 launches of 5-40 us each, and four of them were finishers.
// The partial-sum tensors are kept alive until the launch; flush() runs on the caller's current stream, which must be
// the one their producers ran on.
class FinishQueue {
 public:
  void add(const Tensor& partial, int nblk, int H, int nseg, float* o0, float* o1, float* o2, bool accumulate) {
    if (n_ == PDT_COLSUM_MAX_JOBS) flush();
    keep_.push_back(partial);
    jobs_[n_++] = PdtColsumJob{partial.data_ptr<float>(), {o0, o1, o2, nullptr}, nblk, H, nseg, accumulate ? 1 : 0};
  }
  void flush() {
    if (!n_) return;
    check(pdt_colsum_finish_multi(jobs_, n_, cur_stream()), "colsum_finish_multi");
    n_ = 0;
    keep_.clear();
  }
  // (no flush in the destructor: it would launch, and possibly throw, while an exception unwinds the layer)

 private:
  PdtColsumJob jobs_[PDT_COLSUM_MAX_JOBS];
  int n_ = 0;
  std::vector<Tensor> keep_;
};

struct Epi {
  int kind = PDT_EPI_PLAIN;
  const Tensor* bias = nullptr;
  const Tensor* res = nullptr;
  Tensor* aux = nullptr;
  double drop_p = 0.0;
  PdtRng rng{nullptr, 0, 0};
  Tensor* colsum = nullptr;  // fp32 [N]: (+)= column sums of the stored output (a bias gradient)
  bool colsum_accumulate = true;
  FinishQueue* fq = nullptr;  // the finishing pass of `colsum` is queued here instead of being launched at once
};

void run_gemm(int layout, const Tensor& A, const Tensor& B, Tensor& C, int M, int N, int K, const Epi& e, int tile = -1) {
  PdtGemm g{};
  g.A = A.data_ptr(); g.B = B.data_ptr(); g.C = C.data_ptr();
  g.M = M; g.N = N; g.K = K;
  g.lda = (int)A.stride(0); g.ldb = (int)B.stride(0); g.ldc = (int)C.stride(0);
  g.epi = e.kind;
  if (e.bias) { chk16(*e.bias, "bias"); g.bias = e.bias->data_ptr(); }
  if (e.res) { chk16(*e.res, "res"); g.res = e.res->data_ptr(); g.ldr = (int)e.res->stride(0); }
  if (e.aux) { chk16(*e.aux, "aux"); g.aux = e.aux->data_ptr(); g.ldaux = (int)e.aux->stride(0); }
  g.drop_thr = thr16(e.drop_p);
  g.drop_scale = keep_scale(e.drop_p);
  g.rng = e.rng;
  // column sums: the kernel stores per-wave-row partial sums, a finishing kernel adds them up
  Tensor cs_part;
  if (e.colsum) {
    chkf32(*e.colsum, "colsum");
    TORCH_CHECK(e.colsum->numel() == N, "colsum must have N elements");
    cs_part = at::empty({2 * (((int64_t)M + 63) / 64), (int64_t)N}, C.options().dtype(at::kFloat));
    g.colsum = cs_part.data_ptr<float>();
  }
  // few output tiles + long K: split K over fp32 partial slabs, summed by the epilogue kernel
  Tensor ws;
  const int splits = pdt_gemm_splits(layout, tile, &g);
  if (splits > 1) {
    ws = at::empty({splits, (int64_t)M, (int64_t)N}, C.options().dtype(at::kFloat));
    g.ws = ws.data_ptr<float>();
    g.ws_splits = splits;
  }
  check(pdt_gemm(dt_code(A), layout, tile, &g, cur_stream()), "gemm");
  if (e.colsum && e.fq)
    e.fq->add(cs_part, g.colsum_rows, N, 1, e.colsum->data_ptr<float>(), nullptr, nullptr, e.colsum_accumulate);
  else if (e.colsum)
    check(pdt_colsum_finish(cs_part.data_ptr<float>(), g.colsum_rows, N, 1, e.colsum->data_ptr<float>(), nullptr, nullptr,
                            nullptr, e.colsum_accumulate ? 1 : 0, cur_stream()), "colsum_finish");
}

// C[M,N] = A[M,K] * W[N,K]^T (+ epilogue)
Tensor gemm_nt(const Tensor& A, const Tensor& W, const Epi& e, int tile = -1) {
  chk16(A, "A"); chk16(W, "W");
  const int M = (int)A.size(0), K = (int)A.size(1), N = (int)W.size(0);
  TORCH_CHECK(W.size(1) == K, "gemm_nt: inner dims differ");
  Tensor C = at::empty({M, N}, A.options());
  run_gemm(PDT_GEMM_NT, A, W, C, M, N, K, e, tile);
  return C;
}
// C[M,N] = A[M,K] * W[K,N] (+ epilogue)
Tensor gemm_nn(const Tensor& A, const Tensor& W, const Epi& e, int tile = -1) {
  chk16(A, "A"); chk16(W, "W");
  const int M = (int)A.size(0), K = (int)A.size(1), N = (int)W.size(1);
  TORCH_CHECK(W.size(0) == K, "gemm_nn: inner dims differ");
  Tensor C = at::empty({M, N}, A.options());
  run_gemm(PDT_GEMM_NN, A, W, C, M, N, K, e, tile);
  return C;
}
// G[M,N] (fp32, += when accumulate) = A[K,M]^T * B[K,N]  -- weight gradients; split-K slabs + reduce
void gemm_tn_into(const Tensor& A, const Tensor& B, Tensor& G, bool accumulate, int tile = -1, int splits = 0) {
  chk16(A, "A"); chk16(B, "B"); chkf32(G, "G");
  const int K = (int)A.size(0), M = (int)A.size(1), N = (int)B.size(1);
  TORCH_CHECK(B.size(0) == K && G.size(0) == M && G.size(1) == N, "gemm_tn: shape mismatch");
  // The kernels address an operand through a 32-bit byte offset into a window that, for a weight gradient, spans the
  // whole token range: more than ~2 GiB of either operand (e.g. 262144 tokens x 4096 columns) goes in token chunks,
  // each added to the gradient.
  const int64_t pitch = 2 * std::max<int64_t>(A.stride(0), B.stride(0));
  const int64_t max_rows = ((int64_t)0x7FFF0000 / pitch - 1) / 64 * 64;
  if (K > max_rows) {
    TORCH_CHECK(max_rows >= 64, "gemm_tn: operand rows too long for the 32-bit window");
    for (int64_t k0 = 0; k0 < K; k0 += max_rows) {
      const int64_t len = std::min<int64_t>(max_rows, K - k0);
      gemm_tn_into(A.narrow(0, k0, len), B.narrow(0, k0, len), G, accumulate || k0 > 0, tile, splits);
    }
    return;
  }
  PdtGemm g{};
  g.A = A.data_ptr(); g.B = B.data_ptr();
  g.M = M; g.N = N; g.K = K;
  g.lda = (int)A.stride(0); g.ldb = (int)B.stride(0); g.ldc = N;
  g.epi = PDT_EPI_SLAB_F32;
  g.splits = splits;
  g.splits = pdt_gemm_tn_splits(tile, &g);
  if (g.splits == 1) {  // K is not split: the kernel writes (or adds to) the gradient itself
    g.C = G.data_ptr();
    g.slab_accumulate = accumulate ? 1 : 0;
    check(pdt_gemm(dt_code(A), PDT_GEMM_TN, tile, &g, cur_stream()), "gemm_tn");
    return;
  }
  Tensor slab = at::empty({(int64_t)g.splits * M * N}, G.options());
  g.C = slab.data_ptr();
  check(pdt_gemm(dt_code(A), PDT_GEMM_TN, tile, &g, cur_stream()), "gemm_tn");
  check(pdt_splitk_reduce(slab.data_ptr<float>(), g.splits, (int64_t)M * N, G.data_ptr<float>(), accumulate ? 1 : 0,
                          cur_stream()), "splitk_reduce");
}

// bias gradient of a 16-bit [rows, ncols] matrix into fp32 out[ncols]
void colsum_into(const Tensor& X, Tensor& out, bool accumulate) {
  chk16(X, "X"); chkf32(out, "out");
  const int rows = (int)X.size(0), ncols = (int)X.size(1);
  Tensor partial = at::empty({256, ncols}, out.options());
  int nblk = 0;
  check(pdt_colsum_partial(dt_code(X), X.data_ptr(), rows, ncols, (int)X.stride(0), partial.data_ptr<float>(), &nblk,
                           cur_stream()), "colsum_partial");
  check(pdt_colsum_finish(partial.data_ptr<float>(), nblk, ncols, 1, out.data_ptr<float>(), nullptr, nullptr, nullptr,
                          accumulate ? 1 : 0, cur_stream()), "colsum_finish");
}

struct LnBwdOut { Tensor dx, ddrop; };
// LayerNorm backward + (optional) dropout-masked copy + gamma/beta/bias gradients
LnBwdOut ln_bwd(const Tensor& dy, const Tensor& x, const Tensor& stats, const Tensor& gamma, Tensor* g_gamma,
                Tensor* g_beta, Tensor* g_bias, double drop_p, PdtRng rng, bool accumulate, FinishQueue* fq = nullptr) {
  const int rows = (int)x.size(0), H = (int)x.size(1);
  LnBwdOut o;
  o.dx = at::empty_like(x);
  const bool masked = drop_p > 0.0;
  o.ddrop = masked ? at::empty_like(x) : o.dx;
  Tensor partial = at::empty({(int64_t)pdt_layernorm_bwd_max_blocks() * 3 * H}, stats.options());
  int nblk = 0;
  check(pdt_layernorm_bwd(dt_code(x), dy.data_ptr(), x.data_ptr(), stats.data_ptr<float>(), gamma.data_ptr(),
                          o.dx.data_ptr(), masked ? o.ddrop.data_ptr() : nullptr, partial.data_ptr<float>(), &nblk,
                          rows, H, keep_scale(drop_p), thr16(drop_p), rng, cur_stream()), "layernorm_bwd");
  float* o0 = g_gamma ? g_gamma->data_ptr<float>() : nullptr;
  float* o1 = g_beta ? g_beta->data_ptr<float>() : nullptr;
  float* o2 = g_bias ? g_bias->data_ptr<float>() : nullptr;
  if (fq)
    fq->add(partial, nblk, H, 3, o0, o1, o2, accumulate);
  else
    check(pdt_colsum_finish(partial.data_ptr<float>(), nblk, H, 3, o0, o1, o2, nullptr, accumulate ? 1 : 0, cur_stream()),
          "colsum_finish");
  return o;
}

Tensor ln_fwd(const Tensor& x, const Tensor& gamma, const Tensor& beta, Tensor& stats, double eps) {
  Tensor y = at::empty_like(x);
  check(pdt_layernorm_fwd(dt_code(x), x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(),
                          stats.data_ptr<float>(), (int)x.size(0), (int)x.size(1), (float)eps, cur_stream()),
        "layernorm_fwd");
  return y;
}

// ---------------------------------------------------------------------------------------------------
// Attention with a relative position bias, and the per-head norm + rotation of queries and keys
// ---------------------------------------------------------------------------------------------------
// [B, S, A, D] (or packed [T, A, D]) as the kernels address it; a tensor whose rows they cannot (inner stride other than 1,
// rows off the 16-byte grid, rows too far apart) is copied.
Tensor head_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be 16-bit float");
  bool ok = (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 && (t.size(-1) == 1 || t.stride(-1) == 1);
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= 0 && (i != t.dim() - 3 || t.stride(i) <= (1 << 23))));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// weights, tables, positions and borders as the kernels read them: contiguous and on the 16-byte grid, copied if they are not
OptTensor dense(const OptTensor& t) {
  if (!t.has_value() || (t->is_contiguous() && (!t->has_storage() || (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0))) return t;
  return t->clone(at::MemoryFormat::Contiguous);
}
PdtRelView rel_view(const Tensor& t) {
  const int64_t d = t.dim();
  auto st = [&](int64_t i) { return t.size(i) <= 1 ? (int64_t)0 : t.stride(i); };
  return PdtRelView{t.data_ptr(), d == 4 ? st(0) : 0, st(d - 3), st(d - 2)};
}
// The operators' nodes know the backward pass only.  What else follows a tensor's data - a tangent of forward-mode
// differentiation, a trace that records operations - does not see the kernels and would be lost without a word.
void plain_call(std::initializer_list<const Tensor*> tensors, std::initializer_list<const OptTensor*> more, const char* name) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(Key::PROXY).has_value() && !Modes::get_mode(Key::FAKE).has_value(),
              name, " cannot be traced: a trace would hold its empty output tensor");
  const auto plain = [&](const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name, " has no forward-mode derivative: the tangent would be dropped");
  };
  for (const Tensor* t : tensors) plain(*t);
  for (const OptTensor* t : more)
    if (t->has_value()) plain(**t);
}
void same_gpu(const Tensor& t, const Tensor& as, const char* name) {
  TORCH_CHECK(t.device() == as.device(), name, " must be on the device of q");
}

// What the three kernels of one call share.  q, k, v come from head_rows().  `bits`: int64 mask bits, or the mask itself.
struct RelCall {
  const OptTensor &table, &bits, &cu;
  const std::vector<int64_t>& steps;
  int64_t max_distance, S;
  double scale, p;
};
PdtRelAttn rel_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const RelCall& c, const PdtRng& rng) {
  const bool packed = c.cu.has_value();
  TORCH_CHECK(q.dim() == (packed ? 3 : 4), "q must be ", packed ? "[T, heads, dim] with cu_seqlens" : "[B, S, heads, dim]");
  TORCH_CHECK(k.sizes() == q.sizes() && v.sizes() == q.sizes(), "q, k and v must have one shape (as many key and value heads as query heads)");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have one dtype");
  same_gpu(k, q, "k"); same_gpu(v, q, "v");
  const int64_t D = q.size(-1), A = q.size(-2);
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "the head dim must be a multiple of 8, at most 128 (got ", D, ")");
  TORCH_CHECK(A >= 1, "at least one head");
  PdtRelAttn a{};
  if (packed) {
    TORCH_CHECK(c.cu->scalar_type() == at::kInt && c.cu->is_contiguous() && c.cu->dim() == 1 && c.cu->numel() >= 1,
                "cu_seqlens must be a contiguous int32 [B + 1] tensor");
    same_gpu(*c.cu, q, "cu_seqlens");
    TORCH_CHECK(!c.bits.has_value(), "packed rows take no key mask");
    TORCH_CHECK(q.size(0) <= 0x7FFFFFFF && c.S >= 0 && c.S <= 0x7FFFFFFF, "too many rows");
    TORCH_CHECK(c.S >= 1 || q.size(0) == 0 || c.cu->numel() == 1, "max_seqlen must be at least the longest sequence");
    a.cu = c.cu->data_ptr<int32_t>();
    a.B = (int)c.cu->numel() - 1;
    a.S = (int)std::min<int64_t>(c.S, q.size(0));
    a.T = (int)q.size(0);
  } else {
    a.B = (int)q.size(0); a.S = (int)q.size(1);
    if (c.bits.has_value() && c.bits->scalar_type() != at::kLong) {  // (a mask as key_mask_tensor() leaves it)
      const Tensor& m = *c.bits;
      TORCH_CHECK(m.dim() == 2 && m.size(0) == a.B && m.size(1) == a.S && (a.S <= 1 || m.stride(1) == 1), "key_mask must be [B, S]");
      same_gpu(m, q, "key_mask");
      a.mask = m.data_ptr();
      a.mask_bytes = m.scalar_type() == at::kInt ? 4 : 1;
      a.mask_stride = a.B <= 1 ? 0 : m.stride(0);
    } else if (c.bits.has_value()) {
      TORCH_CHECK(c.bits->scalar_type() == at::kLong && c.bits->is_contiguous() && c.bits->dim() == 2 &&
                  c.bits->size(0) == a.B && c.bits->size(1) == (a.S + 63) / 64, "mask bits must be int64 [B, ceil(S / 64)]");
      same_gpu(*c.bits, q, "mask bits");
      a.mask_bits = reinterpret_cast<const uint64_t*>(c.bits->data_ptr<int64_t>());
      a.mask_words = (int)c.bits->size(1);
    }
  }
  a.A = (int)A; a.D = (int)D;
  a.q = rel_view(q); a.k = rel_view(k); a.v = rel_view(v); a.o = rel_view(o);
  if (c.table.has_value()) {
    const Tensor& t = *c.table;
    same_gpu(t, q, "the bias table");
    TORCH_CHECK(t.dim() == 2 && t.size(1) == A && t.is_contiguous(), "the bias table must be a contiguous [buckets, heads] tensor");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == q.scalar_type(), "the bias table must be fp32 or of q's dtype");
    const int64_t half = t.size(0) / 2;
    TORCH_CHECK((int64_t)c.steps.size() == half - half / 2 && c.steps.size() <= 32, "one step per logarithmic bucket");
    a.table = t.data_ptr();
    a.table_f32 = t.scalar_type() == at::kFloat;
    a.buckets = (int)t.size(0);
    a.max_distance = (int)c.max_distance;
    std::fill(std::begin(a.steps), std::end(a.steps), INT_MAX);
    for (size_t i = 0; i < c.steps.size(); ++i) {
      TORCH_CHECK(c.steps[i] >= (i ? c.steps[i - 1] : half / 2) && c.steps[i] <= c.max_distance, "steps must ascend up to max_distance");
      a.steps[i] = (int)c.steps[i];
    }
  }
  TORCH_CHECK(std::abs(c.scale) >= 0x1p-64 && std::abs(c.scale) <= 0x1p64, "the size of scale must be from 2^-64 to 2^64");
  a.scale = (float)c.scale;
  a.drop_thr = thr16(c.p);
  a.drop_scale = keep_scale(c.p);
  a.rng = rng;
  return a;
}
// key mask [B, S] (bool, uint8 or int32; non-zero = attended) with neighbouring keys
Tensor key_mask_tensor(const Tensor& mask) {
  TORCH_CHECK(mask.is_cuda() && mask.dim() == 2, "the key mask must be a [B, S] GPU tensor");
  const auto st = mask.scalar_type();
  TORCH_CHECK(st == at::kBool || st == at::kByte || st == at::kInt, "the key mask must be bool, uint8 or int32 (non-zero = attended), got ", st);
  TORCH_CHECK(mask.size(0) <= 0x7FFFFFFF && mask.size(1) <= 0x7FFFFFFF, "the key mask is too large");
  return mask.size(1) <= 1 || mask.stride(1) == 1 ? mask : mask.contiguous();
}
// -> one bit per key, int64 [B, ceil(S / 64)]
Tensor rel_mask_bits(const Tensor& mask) {
  const Tensor m = key_mask_tensor(mask);
  DeviceGuard guard(m.device());
  const int64_t B = m.size(0), S = m.size(1);
  Tensor bits = at::empty({B, (S + 63) / 64}, m.options().dtype(at::kLong));
  if (bits.numel())
    check(pdt_rel_attn_mask(m.data_ptr(), m.scalar_type() == at::kInt ? 4 : 1, B <= 1 ? 0 : m.stride(0), (int)B, (int)S,
                            reinterpret_cast<uint64_t*>(bits.data_ptr<int64_t>()), cur_stream()), "rel_attn_mask");
  return bits;
}
PdtRng rel_rng(const OptTensor& state, double p, int64_t micro, int64_t site, const OptTensor& sids, int64_t B, const Tensor& q) {
  if (p <= 0.0 || !state.has_value()) {
    TORCH_CHECK(p <= 0.0, "dropout needs a generator state");
    return PdtRng{nullptr, 0, 0, nullptr, 1u, 0u, nullptr};
  }
  TORCH_CHECK(p <= 0.99, "the dropout probability must be at most 0.99");  // (16-bit probabilities divided by the share kept)
  same_gpu(*state, q, "the generator state");
  if (sids.has_value()) same_gpu(*sids, q, "sample_ids");
  // (the masks derive from (sample, head, query, key): the sequence length plays no part)
  return make_rng(*state, micro, site, sids, 1, B);
}
// log-sum-exps [B, heads, S], or [3, B, heads, S] with the far shares of long rows behind them (PdtRelAttn.mass)
Tensor rel_row_sums(int64_t B, int64_t A, int64_t S, bool table, const at::TensorOptions& f32) {
  return table && pdt_rel_attn_uses_low((int)S) ? at::empty({3, B, A, S}, f32) : at::empty({B, A, S}, f32);
}
void set_row_sums(PdtRelAttn& a, const Tensor& lse) {
  chkf32(lse, "lse");
  const int64_t d = lse.dim() - 3;
  TORCH_CHECK((d == 0 || (d == 1 && lse.size(0) == 3)) && lse.size(d) == a.B && lse.size(d + 1) == a.A && lse.size(d + 2) == a.S,
              "lse must be [B, heads, S] or [3, B, heads, S]");
  a.lse = lse.data_ptr<float>();
  a.mass = d ? a.lse + (int64_t)a.B * a.A * a.S : nullptr;
}
// -> o, lse, o_lo (what a backward pass needs only when wanted; o_lo for long sequences only, see PdtRelAttn)
std::vector<Tensor> rel_attn_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const OptTensor& table,
                                     int64_t max_distance, const std::vector<int64_t>& steps, const OptTensor& bits,
                                     const OptTensor& cu, int64_t max_seqlen, double scale, const OptTensor& rng_state,
                                     double p, int64_t micro, int64_t site, const OptTensor& sids, bool want_lse) {
  TORCH_CHECK(q_in.is_cuda(), "q must be on the GPU");
  DeviceGuard guard(q_in.device());
  const Tensor q = head_rows(q_in, "q"), k = head_rows(k_in, "k"), v = head_rows(v_in, "v");
  Tensor o = at::empty(q.sizes(), q.options());
  const RelCall c{table, bits, cu, steps, max_distance, max_seqlen, scale, p};
  PdtRelAttn a = rel_args(q, k, v, o, c, PdtRng{});
  a.rng = rel_rng(rng_state, p, micro, site, sids, a.B, q);
  if (q.numel() == 0) return {o, want_lse ? at::empty({a.B, a.A, a.S}, q.options().dtype(at::kFloat)) : Tensor(), Tensor()};
  Tensor lse, low;
  if (want_lse) {
    lse = rel_row_sums(a.B, a.A, a.S, table.has_value(), q.options().dtype(at::kFloat));
    set_row_sums(a, lse);
    if (pdt_rel_attn_uses_low(a.S)) {
      low = at::empty(q.sizes(), q.options());
      a.o_lo = rel_view(low);
    }
  }
  if (a.B == 0) o.zero_();  // (rows, but no sequences)
  check(pdt_rel_attn_fwd(dt_code(q), &a, cur_stream()), "rel_attn_fwd");
  return {o, lse, low};
}
// Where a call's parameter gradients go: fp32 (possibly added to what is there), or 16-bit
struct GradOut {
  void* p = nullptr;
  bool half = false, accumulate = false;
};
GradOut grad_out(const Tensor& t) { return t.defined() ? GradOut{t.data_ptr(), t.scalar_type() != at::kFloat, false} : GradOut{}; }
void finish_columns(int dtype, const Tensor& part, int rows, int H, int nseg, const GradOut& a, const GradOut& b) {
  const float* p = rows ? part.data_ptr<float>() : nullptr;
  if (a.half)
    check(pdt_colsum_finish16(dtype, p, rows, H, nseg, a.p, b.p, cur_stream()), "colsum_finish16");
  else
    check(pdt_colsum_finish(p, rows, H, nseg, (float*)a.p, (float*)b.p, nullptr, nullptr, a.accumulate ? 1 : 0, cur_stream()), "colsum_finish");
}
// dq, dk, dv into the given tensors; the table gradient [buckets, A] where `dtable` says
void rel_attn_backward_into(const Tensor& dout_in, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                            const Tensor& low, const Tensor& lse, const RelCall& c, const PdtRng& rng, Tensor dq, Tensor dk, Tensor dv,
                            const GradOut& dtable) {
  PdtRelAttn a = rel_args(q, k, v, o, c, rng);
  const Tensor dout = head_rows(dout_in, "dout");
  TORCH_CHECK(dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type(), "dout must have q's shape and dtype");
  set_row_sums(a, lse);
  Tensor delta = at::empty({2, a.B, a.A, a.S}, lse.options()), part;
  if (low.defined()) {
    TORCH_CHECK(low.sizes() == o.sizes() && low.scalar_type() == o.scalar_type(), "low must have o's shape and dtype");
    a.o_lo = rel_view(low);
  }
  a.dout = rel_view(dout); a.dq = rel_view(dq); a.dk = rel_view(dk); a.dv = rel_view(dv);
  a.delta = delta.data_ptr<float>();
  Tensor peaks;
  if (const int64_t n = pdt_rel_attn_peaks(dt_code(q), &a)) {
    peaks = at::empty({n}, q.options().dtype(at::kInt));
    a.peaks = reinterpret_cast<uint32_t*>(peaks.data_ptr<int32_t>());
  }
  const int rows = pdt_rel_attn_dtable_rows(&a);
  if (dtable.p) {
    part = at::empty({rows, (int64_t)a.buckets * a.A}, lse.options());
    a.dtable_part = part.data_ptr<float>();
  }
  if (a.B == 0)
    for (Tensor t : {dq, dk, dv}) t.zero_();
  check(pdt_rel_attn_bwd(dt_code(q), &a, cur_stream()), "rel_attn_bwd");
  if (dtable.p) finish_columns(dt_code(q), part, rows, a.buckets * a.A, 1, dtable, GradOut{});
}
std::vector<Tensor> rel_attn_backward(const Tensor& dout, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& o,
                                      const Tensor& lse, const OptTensor& low, const OptTensor& table, int64_t max_distance,
                                      const std::vector<int64_t>& steps, const OptTensor& bits, const OptTensor& cu,
                                      int64_t max_seqlen, double scale, const OptTensor& rng_state, double p, int64_t micro,
                                      int64_t site, const OptTensor& sids, bool want_dtable) {
  TORCH_CHECK(q_in.is_cuda(), "q must be on the GPU");
  DeviceGuard guard(q_in.device());
  const Tensor q = head_rows(q_in, "q"), k = head_rows(k_in, "k"), v = head_rows(v_in, "v");
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(q.sizes(), q.options()), dv = at::empty(q.sizes(), q.options());
  Tensor dtable;
  want_dtable = want_dtable && table.has_value();
  if (q.numel() == 0) {
    if (want_dtable) dtable = at::zeros(table->sizes(), table->options());
    return {dq, dk, dv, dtable};
  }
  if (want_dtable) dtable = at::empty(table->sizes(), table->options());
  const RelCall c{table, bits, cu, steps, max_distance, max_seqlen, scale, p};
  rel_attn_backward_into(dout, q, k, v, o, low.has_value() ? *low : Tensor(), lse, c, rel_rng(rng_state, p, micro, site, sids, lse.size(-3), q), dq, dk, dv,
                         grad_out(dtable));
  return {dq, dk, dv, dtable};
}

// The two calls above as one differentiable operation (in C++: a training pass over short packed batches is bound by the
// host, and the Python form of this node cost it 30 us more).
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
struct RelAttnNode : public torch::autograd::Function<RelAttnNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& table,
                        int64_t max_distance, std::vector<int64_t> steps, const OptTensor& bits, const OptTensor& cu,
                        int64_t max_seqlen, double scale, const OptTensor& rng_state, double p, int64_t micro, int64_t site,
                        const OptTensor& sids, bool wanted) {
    std::vector<Tensor> r = rel_attn_forward(q, k, v, table, max_distance, steps, bits, cu, max_seqlen, scale, rng_state, p, micro,
                                             site, sids, wanted);
    if (wanted) {
      auto t = [](const OptTensor& x) { return x.has_value() ? *x : Tensor(); };
      ctx->save_for_backward({q, k, v, t(table), r[0], r[1], t(bits), t(cu), t(rng_state), t(sids), r[2]});
      ctx->saved_data["steps"] = steps;
      ctx->saved_data["ints"] = std::vector<int64_t>{max_distance, max_seqlen, micro, site};
      ctx->saved_data["floats"] = std::vector<double>{scale, p};
    }
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dout) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "relative_attention is not twice differentiable");
    const auto t = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    const auto floats = ctx->saved_data["floats"].toDoubleVector();
    std::vector<Tensor> g = rel_attn_backward(dout[0], t[0], t[1], t[2], t[4], t[5], opt(t[10]), opt(t[3]), ints[0], ctx->saved_data["steps"].toIntVector(),
                                              opt(t[6]), opt(t[7]), ints[1], floats[0], opt(t[8]), floats[1], ints[2], ints[3],
                                              opt(t[9]), t[3].defined() && ctx->needs_input_grad(3));
    torch::autograd::variable_list out(16);
    for (int i = 0; i < 4; ++i) out[i] = g[i];
    return out;
  }
};
// `key_mask`: [B, S] as key_mask_tensor() takes it
Tensor relative_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& table, int64_t max_distance,
                          const std::vector<int64_t>& steps, const OptTensor& key_mask, const OptTensor& cu_in, int64_t max_seqlen,
                          double scale, const OptTensor& rng_state, double p, int64_t micro, int64_t site, const OptTensor& sids) {
  plain_call({&q, &k, &v}, {&table}, "relative_attention");
  TORCH_CHECK(q.is_cuda(), "q must be on the GPU");
  const OptTensor cu = cu_in.has_value() && !cu_in->is_contiguous() ? OptTensor(cu_in->contiguous()) : cu_in;
  OptTensor bits;
  if (key_mask.has_value()) {
    same_gpu(*key_mask, q, "key_mask");
    bits = key_mask->dim() == 2 && key_mask->size(1) <= 128 ? key_mask_tensor(*key_mask) : rel_mask_bits(*key_mask);
  }
  const bool wanted = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                                     (table.has_value() && table->requires_grad()));
  if (!wanted)
    return rel_attn_forward(q, k, v, table, max_distance, steps, bits, cu, max_seqlen, scale, rng_state, p, micro, site, sids, false)[0];
  return RelAttnNode::apply(q, k, v, table, max_distance, steps, bits, cu, max_seqlen, scale, rng_state, p, micro, site, sids, true);
}

// ---- per-head norm + rotation
struct RopeCall {
  const OptTensor &wq, &wk, &cos, &sin, &pos;
  bool interleaved;
  double eps;
};
PdtQkRope rope_args(const Tensor& q, const Tensor& k, const RopeCall& c) {
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be [T, heads, dim] or [B, S, heads, dim]");
  TORCH_CHECK(k.dim() == q.dim() && k.size(0) == q.size(0) && k.size(-1) == q.size(-1) && (q.dim() == 3 || k.size(1) == q.size(1)),
              "q and k must agree in everything but the number of heads");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have one dtype");
  same_gpu(k, q, "k");
  const int64_t D = q.size(-1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "the head dim must be a multiple of 8, at most 256 (got ", D, ")");
  PdtQkRope a{};
  const int64_t T = q.dim() == 4 ? q.size(0) * q.size(1) : q.size(0);
  TORCH_CHECK(T <= (1 << 30), "too many tokens");
  a.T = (int)T;
  a.seq = (int)std::max<int64_t>(1, q.dim() == 4 ? q.size(1) : q.size(0));
  a.D = (int)D;
  a.heads[0] = (int)q.size(-2); a.heads[1] = (int)k.size(-2);
  a.x[0] = rel_view(q); a.x[1] = rel_view(k);
  a.interleaved = c.interleaved;
  a.eps = (float)c.eps;
  const OptTensor* ws[2] = {&c.wq, &c.wk};
  TORCH_CHECK(c.wq.has_value() == c.wk.has_value(), "give both norm weights or neither");
  for (int i = 0; i < 2; ++i) {
    if (!ws[i]->has_value()) continue;
    const Tensor& w = **ws[i];
    same_gpu(w, q, "the norm weights");
    TORCH_CHECK(w.dim() == 1 && w.size(0) == D && w.is_contiguous(), "a norm weight must be a contiguous [dim] tensor");
    TORCH_CHECK(w.scalar_type() == at::kFloat || w.scalar_type() == q.scalar_type(), "norm weights must be fp32 or of q's dtype");
    TORCH_CHECK(w.scalar_type() == c.wq->scalar_type(), "the norm weights must have one dtype");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0, "norm weights must be 16-byte aligned");
    a.w[i] = w.data_ptr();
    a.w_f32 = w.scalar_type() == at::kFloat;
  }
  TORCH_CHECK(!c.wq.has_value() || c.eps > 0.0, "eps must be positive");
  TORCH_CHECK(c.cos.has_value() == c.sin.has_value(), "give cosines and sines");
  if (c.cos.has_value()) {
    chkf32(*c.cos, "cos"); chkf32(*c.sin, "sin");
    same_gpu(*c.cos, q, "cos"); same_gpu(*c.sin, q, "sin");
    TORCH_CHECK(c.cos->dim() == 2 && c.cos->sizes() == c.sin->sizes() && c.cos->size(0) >= 1, "cos and sin must be [positions, rotated / 2]");
    const int64_t R = 2 * c.cos->size(1);
    TORCH_CHECK(R >= 8 && R <= D && R % (c.interleaved ? 8 : 16) == 0, "the rotated part must be a multiple of ", c.interleaved ? 8 : 16,
                " elements, at most the head dim (got ", R, " of ", D, ")");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(c.cos->data_ptr()) & 15) == 0 && (reinterpret_cast<uintptr_t>(c.sin->data_ptr()) & 15) == 0,
                "cos and sin must be 16-byte aligned");
    a.cos = c.cos->data_ptr<float>(); a.sin = c.sin->data_ptr<float>();
    a.R = (int)R;
    a.P = (int)std::min<int64_t>(c.cos->size(0), 0x7FFFFFFF);
    if (c.pos.has_value()) {
      same_gpu(*c.pos, q, "positions");
      TORCH_CHECK(c.pos->scalar_type() == at::kLong && c.pos->is_contiguous() && c.pos->numel() == T, "positions must be a contiguous int64 tensor, one per token");
      a.pos = c.pos->data_ptr<int64_t>();
    } else {
      TORCH_CHECK(a.seq <= c.cos->size(0) || T == 0, "cos and sin have ", c.cos->size(0), " positions, the sequence ", a.seq);
    }
  }
  return a;
}
void rope_forward_into(const Tensor& q, const Tensor& k, const RopeCall& c, Tensor yq, Tensor yk) {
  PdtQkRope a = rope_args(q, k, c);
  a.y[0] = rel_view(yq); a.y[1] = rel_view(yk);
  check(pdt_qk_rope_fwd(dt_code(q), &a, cur_stream()), "qk_rope_fwd");
}
// dxq, dxk into the given tensors; the weight gradients [D] where dwq / dwk say (both or neither)
void rope_backward_into(const Tensor& dyq_in, const Tensor& dyk_in, const Tensor& q, const Tensor& k, const RopeCall& c, Tensor dxq,
                        Tensor dxk, const GradOut& dwq, const GradOut& dwk) {
  PdtQkRope a = rope_args(q, k, c);
  const Tensor dyq = head_rows(dyq_in, "dq"), dyk = head_rows(dyk_in, "dk");
  TORCH_CHECK(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes() && dyq.scalar_type() == q.scalar_type() &&
              dyk.scalar_type() == q.scalar_type(), "gradients must have the shape and dtype of q and k");
  a.y[0] = rel_view(dyq); a.y[1] = rel_view(dyk);
  a.dx[0] = rel_view(dxq); a.dx[1] = rel_view(dxk);
  Tensor part;
  const int blocks = pdt_qk_rope_bwd_blocks(&a);
  if (dwq.p) part = at::empty({blocks, 2 * (int64_t)a.D}, q.options().dtype(at::kFloat));
  check(pdt_qk_rope_bwd(dt_code(q), &a, part.defined() ? part.data_ptr<float>() : nullptr, cur_stream()), "qk_rope_bwd");
  if (part.defined()) finish_columns(dt_code(q), part, blocks, a.D, 2, dwq, dwk);
}
std::vector<Tensor> qk_rope_forward(const Tensor& q_in, const Tensor& k_in, const OptTensor& wq, const OptTensor& wk,
                                    const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, bool interleaved, double eps) {
  TORCH_CHECK(q_in.is_cuda(), "q must be on the GPU");
  DeviceGuard guard(q_in.device());
  const Tensor q = head_rows(q_in, "q"), k = head_rows(k_in, "k");
  Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  rope_forward_into(q, k, RopeCall{wq, wk, cos, sin, pos, interleaved, eps}, yq, yk);
  return {yq, yk};
}
std::vector<Tensor> qk_rope_backward(const Tensor& dyq, const Tensor& dyk, const Tensor& q_in, const Tensor& k_in, const OptTensor& wq,
                                     const OptTensor& wk, const OptTensor& cos, const OptTensor& sin, const OptTensor& pos,
                                     bool interleaved, double eps, bool want_dw) {
  TORCH_CHECK(q_in.is_cuda(), "q must be on the GPU");
  DeviceGuard guard(q_in.device());
  const Tensor q = head_rows(q_in, "q"), k = head_rows(k_in, "k");
  Tensor dxq = at::empty(q.sizes(), q.options()), dxk = at::empty(k.sizes(), k.options()), dwq, dwk;
  if (want_dw && wq.has_value()) {
    dwq = at::empty({q.size(-1)}, wq->options());
    dwk = at::empty({q.size(-1)}, wk->options());
  }
  rope_backward_into(dyq, dyk, q, k, RopeCall{wq, wk, cos, sin, pos, interleaved, eps}, dxq, dxk,
                     grad_out(dwq), grad_out(dwk));
  return {dxq, dxk, dwq, dwk};
}
struct QkRopeNode : public torch::autograd::Function<QkRopeNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const OptTensor& wq, const OptTensor& wk, const OptTensor& cos, const OptTensor& sin,
                                                const OptTensor& pos, bool interleaved, double eps) {
    std::vector<Tensor> y = qk_rope_forward(q, k, wq, wk, cos, sin, pos, interleaved, eps);
    auto t = [](const OptTensor& x) { return x.has_value() ? *x : Tensor(); };
    ctx->save_for_backward({q, k, t(wq), t(wk), t(cos), t(sin), t(pos)});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope is not twice differentiable");
    const auto t = ctx->get_saved_variables();
    const bool want_dw = t[2].defined() && (ctx->needs_input_grad(2) || ctx->needs_input_grad(3));
    std::vector<Tensor> g = qk_rope_backward(dy[0], dy[1], t[0], t[1], opt(t[2]), opt(t[3]), opt(t[4]), opt(t[5]), opt(t[6]),
                                             ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble(), want_dw);
    torch::autograd::variable_list out(9);
    out[0] = g[0];
    out[1] = g[1];
    if (want_dw) {
      out[2] = g[2];
      out[3] = g[3];
    }
    return out;
  }
};
std::vector<Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const OptTensor& wq_in, const OptTensor& wk_in, const OptTensor& cos_in,
                                 const OptTensor& sin_in, const OptTensor& pos_in, bool interleaved, double eps) {
  plain_call({&q, &k}, {&wq_in, &wk_in, &cos_in, &sin_in}, "qk_norm_rope");
  TORCH_CHECK(q.is_cuda(), "q must be on the GPU");
  const OptTensor wq = dense(wq_in), wk = dense(wk_in), cos = dense(cos_in), sin = dense(sin_in), pos = dense(pos_in);
  const bool wanted = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || (wq.has_value() && wq->requires_grad()) ||
                                                     (wk.has_value() && wk->requires_grad()));
  if (!wanted) return qk_rope_forward(q, k, wq, wk, cos, sin, pos, interleaved, eps);
  return QkRopeNode::apply(q, k, wq, wk, cos, sin, pos, interleaved, eps);
}

// ---------------------------------------------------------------------------------------------------
// Encoder layer.  Weight list order (16-bit compute copies):
//   0 wqkv[3H,H] 1 bqkv[3H] 2 wo[H,H] 3 bo[H] 4 ln1_g 5 ln1_b 6 w1[F,H] 7 b1[F] 8 w2[H,F] 9 b2[H] 10 ln2_g 11 ln2_b
// Gradient list: the same order, fp32 views of the gradient arena.
// Saved list: 0 qkv 1 ctx 2 lse 3 z1 4 stats1 5 x1 6 u 7 gact 8 z2 9 stats2, then of a layer with position options the normalised /
// rotated queries and keys [T, 2, A, 64], if it has such, and beyond 128 tokens what rounding took from ctx (PdtRelAttn.o_lo)
// ---------------------------------------------------------------------------------------------------
// What a layer's attention does with positions: a bias table and / or a norm and rotation of its queries and keys.  The
// gradients of `table`, `wq`, `wk` (those that are there) follow the twelve of the gradient list, in this order.
struct LayerPosition {
  OptTensor table, wq, wk, cos, sin;
  int64_t max_distance = 0;
  std::vector<int64_t> steps;
  double eps = 1e-6;
  bool turns() const { return wq.has_value() || cos.has_value(); }
};
using LayerPositionPtr = std::shared_ptr<LayerPosition>;

// thirds of a fused projection [T, 3H] as [B, S, A, 64] (padded) or [T, A, 64] (packed)
Tensor head_third(const Tensor& qkv, int i, int64_t B, int64_t S, int64_t A, bool packed) {
  const Tensor t = qkv.view({qkv.size(0), qkv.size(1) / (A * 64), A, 64}).select(1, i);
  return packed ? t : t.view({B, S, A, 64});
}
Tensor head_view(const Tensor& x, int64_t B, int64_t S, int64_t A, bool packed) {
  return packed ? x.view({x.size(0), A, 64}) : x.view({B, S, A, 64});
}
// attention of a layer with position options: ctx, lse and (where a backward pass wants it) low are filled; returns the normalised /
// rotated queries and keys
Tensor position_attention_forward(const LayerPosition& pos, const Tensor& qkv, Tensor ctx, Tensor lse, const Tensor& low, const OptTensor& positions,
                                  const OptTensor& bits, const OptTensor& cu, int64_t B, int64_t S, int64_t A, double p, const PdtRng& rng) {
  const bool packed = cu.has_value();
  TORCH_CHECK(!packed || !pos.cos.has_value() || positions.has_value(), "packed rows need their positions for the rotation");
  Tensor q = head_third(qkv, 0, B, S, A, packed), k = head_third(qkv, 1, B, S, A, packed), qk;
  const Tensor v = head_third(qkv, 2, B, S, A, packed);
  if (pos.turns()) {
    qk = at::empty({qkv.size(0), 2 * A * 64}, qkv.options());
    const Tensor yq = head_third(qk, 0, B, S, A, packed), yk = head_third(qk, 1, B, S, A, packed);
    rope_forward_into(q, k, RopeCall{pos.wq, pos.wk, pos.cos, pos.sin, positions, false, pos.eps}, yq, yk);
    q = yq; k = yk;
  }
  const Tensor o = head_view(ctx, B, S, A, packed);
  const RelCall c{pos.table, bits, cu, pos.steps, pos.max_distance, S, 0.125, p};
  PdtRelAttn a = rel_args(q, k, v, o, c, rng);
  set_row_sums(a, lse);
  if (low.defined()) a.o_lo = rel_view(head_view(low, B, S, A, packed));
  if (qkv.size(0)) check(pdt_rel_attn_fwd(dt_code(qkv), &a, cur_stream()), "rel_attn_fwd");
  return qk;
}
void position_attention_backward(const LayerPosition& pos, const Tensor& qkv, const Tensor& qk, const Tensor& ctx, const Tensor& low, const Tensor& dctx,
                                 const Tensor& lse, Tensor dqkv, const std::vector<Tensor>& gr, const OptTensor& positions,
                                 const OptTensor& bits, const OptTensor& cu, int64_t B, int64_t S, int64_t A, double p,
                                 const PdtRng& rng, bool accumulate) {
  const bool packed = cu.has_value();
  auto third = [&](const Tensor& t, int i) { return head_third(t, i, B, S, A, packed); };
  const bool turns = pos.turns();
  TORCH_CHECK((int)gr.size() == 12 + (pos.table.has_value() ? 1 : 0) + (pos.wq.has_value() ? 2 : 0), "layer_backward: gradients of the position parameters missing");
  size_t at = 12;
  auto grad = [&](bool there) { return there ? GradOut{gr[at++].data_ptr<float>(), false, accumulate} : GradOut{}; };
  const GradOut dtable = grad(pos.table.has_value()), dwq = grad(pos.wq.has_value()), dwk = grad(pos.wq.has_value());
  const RelCall c{pos.table, bits, cu, pos.steps, pos.max_distance, S, 0.125, p};
  const Tensor dqk = turns ? at::empty_like(qk) : dqkv;
  rel_attn_backward_into(head_view(dctx, B, S, A, packed), third(turns ? qk : qkv, 0), third(turns ? qk : qkv, 1), third(qkv, 2),
                         head_view(ctx, B, S, A, packed), low.defined() ? head_view(low, B, S, A, packed) : Tensor(), lse, c, rng, third(dqk, 0), third(dqk, 1), third(dqkv, 2), dtable);
  if (turns)
    rope_backward_into(third(dqk, 0), third(dqk, 1), third(qkv, 0), third(qkv, 1),
                       RopeCall{pos.wq, pos.wk, pos.cos, pos.sin, positions, false, pos.eps}, third(dqkv, 0), third(dqkv, 1), dwq, dwk);
}
struct LayerDims { int B, S, A; double p_attn, p_hidden, eps; int64_t micro, layer; };

std::vector<Tensor> layer_forward(const Tensor& x, const Tensor& mask, const Tensor& kv_len,
                                  const std::vector<Tensor>& w, const Tensor& rng_state, int64_t B, int64_t S, int64_t A,
                                  double p_attn, double p_hidden, double eps, int64_t micro, int64_t layer,
                                  const OptTensor& sids, const OptTensor& cu, const OptTensor& rowmap,
                                  const LayerPositionPtr& pos, const OptTensor& positions, const OptTensor& bits, bool tape) {
  DeviceGuard guard(x.device());
  chk16(x, "x");
  TORCH_CHECK(w.size() == 12, "layer_forward: 12 weight tensors expected");
  const int T = (int)x.size(0), H = (int)x.size(1);
  // unpadded batch: x is the packed [T, H] of B samples whose first rows are cu[0..B) (cu[B] = T), S the longest one
  const int32_t* cup = nullptr;
  if (cu.has_value()) {
    TORCH_CHECK(cu->is_cuda() && cu->scalar_type() == at::kInt && cu->is_contiguous() && cu->numel() == B + 1,
                "cu_seqlens must be a contiguous int32 [B+1] GPU tensor");
    TORCH_CHECK(rowmap.has_value() && rowmap->numel() == T, "an unpadded batch needs the per-row dropout table");
    TORCH_CHECK(T <= B * S && H == A * 64, "layer_forward: packed x has more rows than B * S");
    cup = cu->data_ptr<int32_t>();
  } else {
    TORCH_CHECK(T == B * S && H == A * 64, "layer_forward: head_dim must be 64 and x must be [B*S, H]");
  }
  auto f32 = x.options().dtype(at::kFloat);
  const int64_t site = layer * 4;

  Epi e_bias; e_bias.kind = PDT_EPI_BIAS; e_bias.bias = &w[1];
  Tensor qkv = gemm_nt(x, w[0], e_bias);

  Tensor ctx = at::empty({T, H}, x.options());
  Tensor qk, low;
  // (the position kernels count packed rows by the longest sample there can be: no more than the rows there are)
  const int64_t longest = cup ? std::min<int64_t>(S, T) : S;
  Tensor lse = pos ? rel_row_sums(B, A, longest, pos->table.has_value(), f32) : at::empty({B, A, S}, f32);
  if (pos && tape && pdt_rel_attn_uses_low((int)longest)) low = at::empty({T, H}, x.options());
  if (pos)
    qk = position_attention_forward(*pos, qkv, ctx, lse, low, positions, bits, cu, B, S, A, p_attn,
                                    make_rng(rng_state, micro, site + 0, sids, S, B));
  else
    check(pdt_attn_fwd(dt_code(x), qkv.data_ptr(), mask.data_ptr<int32_t>(), kv_len.data_ptr<int32_t>(), cup, ctx.data_ptr(),
                       lse.data_ptr<float>(), (int)B, (int)S, (int)A, keep_scale(p_attn), thr16(p_attn),
                       make_rng(rng_state, micro, site + 0, sids, S, B), cur_stream()), "attn_fwd");

  Epi e_ao; e_ao.kind = PDT_EPI_BIAS_DROP_RES; e_ao.bias = &w[3]; e_ao.res = &x; e_ao.drop_p = p_hidden;
  e_ao.rng = make_rng(rng_state, micro, site + 1, sids, S, B, rowmap);
  Tensor z1 = gemm_nt(ctx, w[2], e_ao);
  Tensor stats1 = at::empty({T, 2}, f32);
  Tensor x1 = ln_fwd(z1, w[4], w[5], stats1, eps);

  Tensor u = at::empty({T, (int64_t)w[6].size(0)}, x.options());  // gelu'(FFN1 pre-activation), for backward
  Epi e_f1; e_f1.kind = PDT_EPI_BIAS_GELU; e_f1.bias = &w[7]; e_f1.aux = &u;
  Tensor gact = gemm_nt(x1, w[6], e_f1);

  Epi e_f2; e_f2.kind = PDT_EPI_BIAS_DROP_RES; e_f2.bias = &w[9]; e_f2.res = &x1; e_f2.drop_p = p_hidden;
  e_f2.rng = make_rng(rng_state, micro, site + 2, sids, S, B, rowmap);
  Tensor z2 = gemm_nt(gact, w[8], e_f2);
  Tensor stats2 = at::empty({T, 2}, f32);
  Tensor x2 = ln_fwd(z2, w[10], w[11], stats2, eps);
  std::vector<Tensor> out = {x2, qkv, ctx, lse, z1, stats1, x1, u, gact, z2, stats2};
  if (qk.defined()) out.push_back(qk);
  if (low.defined()) out.push_back(low);
  return out;
}

Tensor layer_backward(const Tensor& dy_in, const Tensor& x, const std::vector<Tensor>& sv, const Tensor& mask,
                      const Tensor& kv_len, const std::vector<Tensor>& w, std::vector<Tensor> gr,
                      const Tensor& rng_state, int64_t B, int64_t S, int64_t A, double p_attn, double p_hidden,
                      int64_t micro, int64_t layer, bool accumulate, const OptTensor& sids, const OptTensor& cu,
                      const OptTensor& rowmap, const LayerPositionPtr& pos, const OptTensor& positions, const OptTensor& bits) {
  DeviceGuard guard(x.device());
  const int32_t* cup = cu.has_value() ? cu->data_ptr<int32_t>() : nullptr;
  const size_t turns = pos && pos->turns(), lows = pos && pdt_rel_attn_uses_low((int)(cup ? std::min<int64_t>(S, x.size(0)) : S));
  TORCH_CHECK(sv.size() == 10 + turns + lows && w.size() == 12 && (pos || gr.size() == 12), "layer_backward: bad list sizes");
  const Tensor dy = dy_in.contiguous();
  chk16(dy, "dy");
  const Tensor &qkv = sv[0], &ctx = sv[1], &lse = sv[2], &z1 = sv[3], &stats1 = sv[4], &x1 = sv[5], &u = sv[6],
               &gact = sv[7], &z2 = sv[8], &stats2 = sv[9];
  const int T = (int)x.size(0), H = (int)x.size(1);
  const int64_t site = layer * 4;

  FinishQueue fq;  // the four column-sum finishers of the layer run as one launch at its end
  // LN2 -> dz2 (residual path) and ddrop2 (through the FFN2 output dropout); d gamma/beta/b2
  LnBwdOut l2 = ln_bwd(dy, z2, stats2, w[10], &gr[10], &gr[11], &gr[9], p_hidden, make_rng(rng_state, micro, site + 2, sids, S, B, rowmap),
                       accumulate, &fq);
  // FFN2 dgrad fused with GELU' and with the FFN1 bias gradient (column sums of dU) ; wgrad
  Epi e_dg; e_dg.kind = PDT_EPI_MUL_DGELU; e_dg.aux = const_cast<Tensor*>(&u);
  e_dg.colsum = &gr[7]; e_dg.colsum_accumulate = accumulate; e_dg.fq = &fq;
  WgradLane lane(g_wgrad_mode == 2 || (g_wgrad_mode == 1 && T <= kWgradLaneMaxTokens), g_wgrad_defer);
  lane.run([&] { gemm_tn_into(l2.ddrop, gact, gr[8], accumulate); }, {l2.ddrop, gact});
  Tensor du = gemm_nn(l2.ddrop, w[8], e_dg);
  // FFN1 dgrad + residual gradient ; wgrad
  Epi e_add; e_add.kind = PDT_EPI_ADD_RES; e_add.res = &l2.dx;
  lane.run([&] { gemm_tn_into(du, x1, gr[6], accumulate); }, {du, x1});
  Tensor dx1 = gemm_nn(du, w[6], e_add);
  // LN1
  LnBwdOut l1 = ln_bwd(dx1, z1, stats1, w[4], &gr[4], &gr[5], &gr[3], p_hidden, make_rng(rng_state, micro, site + 1, sids, S, B, rowmap),
                       accumulate, &fq);
  // attention output projection
  lane.run([&] { gemm_tn_into(l1.ddrop, ctx, gr[2], accumulate); }, {l1.ddrop, ctx});
  Tensor dctx = gemm_nn(l1.ddrop, w[2], Epi{});
  // attention core
  Tensor dqkv = at::empty_like(qkv);
  Tensor delta = at::empty_like(lse);
  // the short-sequence backward kernel also emits per-sample column sums of dqkv (the QKV bias gradient)
  const bool fused_db = !pos && pdt_attn_bwd_fuses_dbias((int)S) != 0;
  const int db_rows = pdt_attn_bwd_dbias_rows((int)B, (int)S);
  Tensor db_part = fused_db ? at::empty({(int64_t)db_rows, 3 * (int64_t)H}, lse.options()) : Tensor();
  if (pos)
    position_attention_backward(*pos, qkv, turns ? sv[10] : Tensor(), ctx, lows ? sv[10 + turns] : Tensor(), dctx, lse, dqkv, gr, positions, bits, cu, B, S, A,
                                p_attn, make_rng(rng_state, micro, site + 0, sids, S, B), accumulate);
  else
    check(pdt_attn_bwd(dt_code(x), qkv.data_ptr(), mask.data_ptr<int32_t>(), kv_len.data_ptr<int32_t>(), cup, ctx.data_ptr(),
                     dctx.data_ptr(), lse.data_ptr<float>(), delta.data_ptr<float>(), dqkv.data_ptr(),
                     fused_db ? db_part.data_ptr<float>() : nullptr, (int)B, (int)S, (int)A, keep_scale(p_attn),
                     thr16(p_attn), make_rng(rng_state, micro, site + 0, sids, S, B), cur_stream()),
        "attn_bwd");
  if (fused_db)
    fq.add(db_part, db_rows, 3 * H, 1, gr[1].data_ptr<float>(), nullptr, nullptr, accumulate);
  else
    colsum_into(dqkv, gr[1], accumulate);
  // QKV projection dgrad + residual gradient ; wgrad
  Epi e_add2; e_add2.kind = PDT_EPI_ADD_RES; e_add2.res = &l1.dx;
  lane.run([&] { gemm_tn_into(dqkv, x, gr[0], accumulate); }, {dqkv, x});
  Tensor dx = gemm_nn(dqkv, w[0], e_add2);
  fq.flush();
  // the layer's gradients are complete on the main stream from here (bucket all-reduce, next layer) - or, deferred,
  // once the caller has joined after the backward pass
  lane.finish();
  (void)T; (void)H;
  return dx;
}

// ---------------------------------------------------------------------------------------------------
// A run of encoder layers as ONE call (one autograd node per stack instead of one per layer): with short
// micro-batches the host, not the GPU, bounds a step, and the Python / autograd round trip per layer is a fifth
// of the host time of a layer.  `layer_ids`: dropout site base of every layer.  Forward returns, per layer, the 11
// tensors of layer_forward (output first); the input of layer l > 0 is the output of layer l-1.
// ---------------------------------------------------------------------------------------------------
std::vector<Tensor> stack_forward(const Tensor& x, const Tensor& mask, const Tensor& kv_len,
                                  const std::vector<std::vector<Tensor>>& w, const Tensor& rng_state, int64_t B, int64_t S,
                                  int64_t A, double p_attn, double p_hidden, double eps, int64_t micro,
                                  const std::vector<int64_t>& layer_ids, const OptTensor& sids, const OptTensor& cu,
                                  const OptTensor& rowmap, const std::vector<LayerPositionPtr>& pos, const OptTensor& positions,
                                  const OptTensor& bits) {
  TORCH_CHECK(!w.empty() && w.size() == layer_ids.size() && pos.size() == w.size(), "stack_forward: one weight list and one id per layer");
  std::vector<Tensor> all;
  all.reserve(w.size() * 13);
  Tensor h = x;
  for (size_t l = 0; l < w.size(); ++l) {
    std::vector<Tensor> o = layer_forward(h, mask, kv_len, w[l], rng_state, B, S, A, p_attn, p_hidden, eps, micro,
                                          layer_ids[l], sids, cu, rowmap, pos[l], positions, bits, true);
    h = o[0];
    for (auto& t : o) all.push_back(std::move(t));
  }
  return all;
}

// Backward of the run, last layer first.  `saved[l]` = the 11 to 13 tensors stack_forward returned for layer l;
// `accumulate[l]`: add to layer l's gradients instead of overwriting them.  After every layer its saved tensors
// are dropped and `layer_done(l)` is called with the GIL held (the Python side drops ITS references there and
// reports the layer's gradient segment as complete: bucket all-reduce, gradient-lane merge).
Tensor stack_backward(const Tensor& dy_in, const Tensor& x0, std::vector<std::vector<Tensor>> saved, const Tensor& mask,
                      const Tensor& kv_len, const std::vector<std::vector<Tensor>>& w,
                      const std::vector<std::vector<Tensor>>& gr, const Tensor& rng_state, int64_t B, int64_t S, int64_t A,
                      double p_attn, double p_hidden, int64_t micro, const std::vector<int64_t>& layer_ids,
                      const std::vector<int64_t>& accumulate, const OptTensor& sids, const OptTensor& cu,
                      const OptTensor& rowmap, py::handle layer_done, const std::vector<LayerPositionPtr>& pos,
                      const OptTensor& positions, const OptTensor& bits) {
  const size_t L = w.size();
  TORCH_CHECK(L > 0 && saved.size() == L && gr.size() == L && layer_ids.size() == L && accumulate.size() == L && pos.size() == L,
              "stack_backward: per-layer lists of different lengths");
  Tensor dy = dy_in;
  for (size_t i = L; i-- > 0;) {
    TORCH_CHECK(saved[i].size() >= 11, "stack_backward: 11 saved tensors per layer expected");
    const Tensor& xin = i == 0 ? x0 : saved[i - 1][0];
    std::vector<Tensor> sv(saved[i].begin() + 1, saved[i].end());
    dy = layer_backward(dy, xin, sv, mask, kv_len, w[i], gr[i], rng_state, B, S, A, p_attn, p_hidden, micro, layer_ids[i],
                        accumulate[i] != 0, sids, cu, rowmap, pos[i], positions, bits);
    sv.clear();
    saved[i].clear();
    if (!layer_done.is_none()) {
      py::gil_scoped_acquire gil;
      layer_done((int64_t)i);
    }
  }
  return dy;
}

// ---------------------------------------------------------------------------------------------------
// Embeddings
// ---------------------------------------------------------------------------------------------------
std::vector<Tensor> embed_forward(const c10::optional<Tensor>& ids, const Tensor& pos_ids, const Tensor& type_ids,
                                  const c10::optional<Tensor>& inputs_embeds, const Tensor& word, const Tensor& pos,
                                  const Tensor& type, const Tensor& gamma, const Tensor& beta, const Tensor& rng_state,
                                  double eps, double p, int64_t micro, int64_t site, const OptTensor& sids, int64_t seq,
                                  const OptTensor& rowmap) {
  DeviceGuard guard(word.device());
  const int H = (int)word.size(1);
  const int tokens = (int)pos_ids.numel();
  TORCH_CHECK(rowmap.has_value() || (seq >= 1 && tokens % seq == 0),
              "embed_forward: tokens must be a multiple of the sequence length");
  const OptTensor no_ids;
  const OptTensor& rsids = rowmap.has_value() ? no_ids : sids;  // (packed rows: the table alone defines the dropout rows)
  const int64_t rbatch = rowmap.has_value() ? -1 : tokens / seq;
  Tensor pre = at::empty({tokens, H}, word.options());
  Tensor y = at::empty({tokens, H}, word.options());
  Tensor stats = at::empty({tokens, 2}, word.options().dtype(at::kFloat));
  const int64_t* idp = ids.has_value() ? ids->data_ptr<int64_t>() : nullptr;
  const void* iep = nullptr;
  if (inputs_embeds.has_value()) { chk16(*inputs_embeds, "inputs_embeds"); iep = inputs_embeds->data_ptr(); }
  check(pdt_embed_fwd(dt_code(word), idp, pos_ids.data_ptr<int64_t>(), type_ids.data_ptr<int64_t>(), iep,
                      word.data_ptr(), pos.data_ptr(), type.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
                      pre.data_ptr(), y.data_ptr(), stats.data_ptr<float>(), tokens, H, (int)word.size(0), (int)pos.size(0),
                      (int)type.size(0), (float)eps, keep_scale(p),
                      thr16(p), make_rng(rng_state, micro, site, rsids, seq, rbatch, rowmap), cur_stream()), "embed_fwd");
  return {y, pre, stats};
}

// grads order: 0 word 1 pos 2 type 3 gamma 4 beta (fp32 arena views).  Returns the gradient wrt the summed
// embedding (needed only when the caller fed inputs_embeds and wants its gradient).
Tensor embed_backward(const Tensor& dy_in, const Tensor& pre, const Tensor& stats, const c10::optional<Tensor>& ids,
                      const Tensor& pos_ids, const Tensor& type_ids, const Tensor& gamma, std::vector<Tensor> gr,
                      const Tensor& rng_state, double p, int64_t micro, int64_t site, int64_t pad_id, bool accumulate,
                      const OptTensor& sids, int64_t seq, const OptTensor& rowmap) {
  DeviceGuard guard(pre.device());
  const OptTensor no_ids;
  const OptTensor& rsids = rowmap.has_value() ? no_ids : sids;
  TORCH_CHECK(gr.size() == 5, "embed_backward: 5 gradient tensors expected");
  const Tensor dy = dy_in.contiguous();
  const int tokens = (int)pre.size(0), H = (int)pre.size(1);
  Tensor dmask = dy;
  if (p > 0.0) {
    dmask = at::empty_like(dy);
    check(pdt_dropout_apply(dt_code(dy), dy.data_ptr(), dmask.data_ptr(), dy.numel(), H, keep_scale(p), thr16(p),
                            make_rng(rng_state, micro, site, rsids, seq, rowmap.has_value() ? -1 : tokens / seq, rowmap),
                            cur_stream()), "dropout_apply");
  }
  LnBwdOut l = ln_bwd(dmask, pre, stats, gamma, &gr[3], &gr[4], nullptr, 0.0, make_rng(rng_state, micro, site),
                      accumulate);
  if (!accumulate) {
    gr[0].zero_();
    gr[1].zero_();
  }
  // word / position tables: sort the indices once (stable: equal indices keep their token order), then the
  // segmented-sum kernels add every run of equal indices to its row - deterministic, no atomics
  auto scatter = [&](const Tensor& idx, Tensor& table, int64_t skip) {
    auto sorted_perm = at::sort(idx, /*stable=*/true, /*dim=*/0, /*descending=*/false);
    const Tensor& sorted = std::get<0>(sorted_perm);
    const Tensor& perm = std::get<1>(sorted_perm);
    Tensor scratch = at::empty({(int64_t)pdt_embed_seg_chunks(tokens) * 2 * H}, stats.options());
    check(pdt_embed_scatter_sorted(dt_code(pre), l.dx.data_ptr(), sorted.data_ptr<int64_t>(), perm.data_ptr<int64_t>(),
                                   table.data_ptr<float>(), scratch.data_ptr<float>(), tokens, H, (int)table.size(0), skip,
                                   cur_stream()), "embed_scatter_sorted");
  };
  if (ids.has_value()) scatter(*ids, gr[0], pad_id);
  scatter(pos_ids, gr[1], -1);
  const int R = (int)gr[2].size(0);
  Tensor partial = at::empty({256, R, H}, stats.options());
  int nblk = 0;
  check(pdt_embed_type_partial(dt_code(pre), l.dx.data_ptr(), type_ids.data_ptr<int64_t>(), partial.data_ptr<float>(),
                               &nblk, tokens, H, R, cur_stream()), "embed_type_partial");
  float* gt = gr[2].data_ptr<float>();
  check(pdt_colsum_finish(partial.data_ptr<float>(), nblk, H, R, gt, R > 1 ? gt + H : nullptr,
                          R > 2 ? gt + 2 * H : nullptr, R > 3 ? gt + 3 * H : nullptr, accumulate ? 1 : 0, cur_stream()),
        "colsum_finish");
  return l.dx;
}

// ---------------------------------------------------------------------------------------------------
// Pooler (dense + tanh on token 0) and classifier + cross-entropy
// ---------------------------------------------------------------------------------------------------
Tensor dense_tanh_forward(const Tensor& first_tok, const Tensor& W, const Tensor& bias) {
  DeviceGuard guard(W.device());
  Epi e; e.kind = PDT_EPI_BIAS_TANH; e.bias = &bias;
  return gemm_nt(first_tok, W, e, 0);
}
// dfirst = dpre * W ; gW += dpre^T * first ; gb += colsum(dpre)     (dpre = grad wrt the pre-tanh value)
Tensor dense_backward(const Tensor& dpre, const Tensor& first_tok, const Tensor& W, Tensor gW, Tensor gb, bool accumulate) {
  DeviceGuard guard(W.device());
  Tensor dfirst = gemm_nn(dpre, W, Epi{}, 0);
  gemm_tn_into(dpre, first_tok, gW, accumulate, 0);
  colsum_into(dpre, gb, accumulate);
  return dfirst;
}

std::vector<Tensor> head_forward(const Tensor& pooled, const Tensor& W, const Tensor& bias,
                                 const c10::optional<Tensor>& labels, const Tensor& rng_state, double p, int64_t micro,
                                 int64_t site, const OptTensor& sids) {
  DeviceGuard guard(pooled.device());
  chk16(pooled, "pooled"); chkf32(W, "W"); chkf32(bias, "bias");
  const int B = (int)pooled.size(0), H = (int)pooled.size(1), C = (int)W.size(0);
  TORCH_CHECK(pooled.is_contiguous(), "pooled must be contiguous");
  if (labels.has_value())
    TORCH_CHECK(labels->is_contiguous() && labels->scalar_type() == at::kLong && labels->numel() == B,
                "labels must be a contiguous int64 [B] tensor");
  auto f32 = W.options();
  Tensor logits = at::empty({B, C}, f32);
  Tensor loss = at::zeros({}, f32);
  check(pdt_head_fwd(dt_code(pooled), pooled.data_ptr(), W.data_ptr<float>(), bias.data_ptr<float>(),
                     labels.has_value() ? labels->data_ptr<int64_t>() : nullptr, logits.data_ptr<float>(),
                     loss.data_ptr<float>(), B, H, C, keep_scale(p), thr16(p), make_rng(rng_state, micro, site, sids, 1, B),
                     cur_stream()), "head_fwd");
  return {logits, loss};
}

Tensor head_backward(const c10::optional<Tensor>& gloss, const c10::optional<Tensor>& dlogits, const Tensor& pooled,
                     const Tensor& W, const Tensor& logits, const c10::optional<Tensor>& labels, Tensor gW, Tensor gb,
                     const Tensor& rng_state, double p, int64_t micro, int64_t site, bool accumulate, bool tanh_bwd,
                     const OptTensor& sids) {
  DeviceGuard guard(pooled.device());
  const int B = (int)pooled.size(0), H = (int)pooled.size(1), C = (int)W.size(0);
  Tensor gl, dl;
  const bool ce = gloss.has_value() && labels.has_value();
  if (ce) gl = gloss->to(at::kFloat).contiguous();
  if (dlogits.has_value()) dl = dlogits->to(at::kFloat).contiguous();
  Tensor dpooled = at::empty_like(pooled);
  const int64_t ws_n = pdt_head_bwd_ws_floats(B, H, C);
  Tensor ws = ws_n > 0 ? at::empty({ws_n}, gW.options()) : Tensor();
  check(pdt_head_bwd(dt_code(pooled), pooled.data_ptr(), W.data_ptr<float>(), logits.data_ptr<float>(),
                     ce ? labels->data_ptr<int64_t>() : nullptr, ce ? gl.data_ptr<float>() : nullptr,
                     dl.defined() ? dl.data_ptr<float>() : nullptr, dpooled.data_ptr(), gW.data_ptr<float>(),
                     gb.data_ptr<float>(), B, H, C, keep_scale(p), thr16(p), make_rng(rng_state, micro, site, sids, 1, B),
                     accumulate ? 1 : 0, tanh_bwd ? 1 : 0, ws_n > 0 ? ws.data_ptr<float>() : nullptr, cur_stream()), "head_bwd");
  return dpooled;
}

// x: [B, H] (one row per sample)
Tensor dropout16(const Tensor& x, const Tensor& rng_state, double p, int64_t micro, int64_t site, const OptTensor& sids) {
  DeviceGuard guard(x.device());
  Tensor xc = x.contiguous();
  Tensor y = at::empty_like(xc);
  TORCH_CHECK(xc.dim() == 2, "dropout16 expects a [B, H] tensor");
  check(pdt_dropout_apply(dt_code(xc), xc.data_ptr(), y.data_ptr(), xc.numel(), (int)xc.size(1), keep_scale(p), thr16(p),
                          make_rng(rng_state, micro, site, sids, 1, xc.size(0)), cur_stream()), "dropout_apply");
  return y;
}

// ---------------------------------------------------------------------------------------------------
// Optimizer
// ---------------------------------------------------------------------------------------------------
void adamw_step(Tensor p, Tensor m, Tensor v, const Tensor& g, const c10::optional<Tensor>& p16, const Tensor& lr,
                const Tensor& step, Tensor scale_state, double beta1, double beta2, double eps, double weight_decay,
                bool correct_bias, bool check_finite) {
  DeviceGuard guard(p.device());
  chkf32(p, "p"); chkf32(m, "m"); chkf32(v, "v"); chkf32(g, "g"); chkf32(lr, "lr"); chkf32(scale_state, "scale_state");
  TORCH_CHECK(step.scalar_type() == at::kInt && step.is_cuda(), "step must be an int32 GPU scalar");
  TORCH_CHECK(scale_state.numel() >= 4, "scale_state: float[4]");
  if (check_finite) check(pdt_grad_check(g.data_ptr<float>(), g.numel(), scale_state.data_ptr<float>(), cur_stream()), "grad_check");
  PdtAdamW a{};
  a.p = p.data_ptr<float>(); a.m = m.data_ptr<float>(); a.v = v.data_ptr<float>(); a.g = g.data_ptr<float>();
  int dtype = PDT_F16;
  if (p16.has_value()) { chk16(*p16, "p16"); a.p16 = p16->data_ptr(); dtype = dt_code(*p16); }
  a.n = p.numel();
  a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.eps = (float)eps; a.weight_decay = (float)weight_decay;
  a.correct_bias = correct_bias ? 1 : 0;
  a.lr = lr.data_ptr<float>(); a.step = step.data_ptr<int32_t>(); a.scale_state = scale_state.data_ptr<float>();
  check(pdt_adamw_step(dtype, &a, cur_stream()), "adamw_step");
}
void grad_check(const Tensor& g, Tensor scale_state) {
  DeviceGuard guard(g.device());
  chkf32(g, "g");
  check(pdt_grad_check(g.data_ptr<float>(), g.numel(), scale_state.data_ptr<float>(), cur_stream()), "grad_check");
}
void scaler_update(Tensor scale_state, Tensor step, double growth, double backoff, int64_t interval, bool dynamic) {
  DeviceGuard guard(scale_state.device());
  check(pdt_scaler_update(scale_state.data_ptr<float>(), step.data_ptr<int32_t>(), (float)growth, (float)backoff,
                          (int)interval, dynamic ? 1 : 0, cur_stream()), "scaler_update");
}
void cast_to_16(const Tensor& src, Tensor dst) {
  DeviceGuard guard(src.device());
  chkf32(src, "src"); chk16(dst, "dst");
  TORCH_CHECK(src.numel() == dst.numel(), "cast_to_16: size mismatch");
  check(pdt_cast_f32_to_16(dt_code(dst), src.data_ptr<float>(), dst.data_ptr(), src.numel(), cur_stream()), "cast");
}

// ---------------------------------------------------------------------------------------------------
// Single-op entry points (unit tests, micro-benchmarks)
// ---------------------------------------------------------------------------------------------------
Tensor op_gemm(const std::string& layout, const Tensor& A, const Tensor& B, int64_t epi,
               const c10::optional<Tensor>& bias, const c10::optional<Tensor>& res, c10::optional<Tensor> aux,
               const c10::optional<Tensor>& rng_state, double drop_p, int64_t micro, int64_t site, int64_t tile,
               c10::optional<Tensor> colsum, const OptTensor& sids, int64_t seq) {
  DeviceGuard guard(A.device());
  Epi e; e.kind = (int)epi; e.drop_p = drop_p;
  if (colsum.has_value()) e.colsum = &*colsum;  // adds to the tensor's content
  if (bias.has_value()) e.bias = &*bias;
  if (res.has_value()) e.res = &*res;
  if (aux.has_value()) e.aux = &*aux;
  if (rng_state.has_value()) e.rng = make_rng(*rng_state, micro, site, sids, seq, sids.has_value() ? A.size(0) / seq : -1);
  if (layout == "nt") return gemm_nt(A, B, e, (int)tile);
  if (layout == "nn") return gemm_nn(A, B, e, (int)tile);
  TORCH_CHECK(false, "op_gemm: layout must be nt or nn");
}
Tensor op_gemm_tn(const Tensor& A, const Tensor& B, c10::optional<Tensor> into, bool accumulate, int64_t tile, int64_t splits) {
  DeviceGuard guard(A.device());
  Tensor G = into.has_value() ? *into : at::zeros({A.size(1), B.size(1)}, A.options().dtype(at::kFloat));
  gemm_tn_into(A, B, G, accumulate, (int)tile, (int)splits);
  return G;
}
std::vector<Tensor> op_layernorm_fwd(const Tensor& x, const Tensor& gamma, const Tensor& beta, double eps) {
  DeviceGuard guard(x.device());
  chk16(x, "x");
  Tensor stats = at::empty({x.size(0), 2}, x.options().dtype(at::kFloat));
  Tensor y = ln_fwd(x, gamma, beta, stats, eps);
  return {y, stats};
}
std::vector<Tensor> op_layernorm_bwd(const Tensor& dy, const Tensor& x, const Tensor& stats, const Tensor& gamma,
                                     const c10::optional<Tensor>& rng_state, double drop_p, int64_t micro, int64_t site,
                                     const OptTensor& sids, int64_t seq) {
  DeviceGuard guard(x.device());
  const int H = (int)x.size(1);
  auto f32 = stats.options();
  Tensor gg = at::zeros({H}, f32), gb = at::zeros({H}, f32), gbias = at::zeros({H}, f32);
  PdtRng rng{nullptr, 0, 0};
  if (rng_state.has_value()) rng = make_rng(*rng_state, micro, site, sids, seq, sids.has_value() ? x.size(0) / seq : -1);
  LnBwdOut o = ln_bwd(dy.contiguous(), x, stats, gamma, &gg, &gb, &gbias, drop_p, rng, false);
  return {o.dx, o.ddrop, gg, gb, gbias};
}
std::vector<Tensor> op_attn_fwd(const Tensor& qkv, const Tensor& mask, const Tensor& kv_len, int64_t B, int64_t S, int64_t A,
                                const c10::optional<Tensor>& rng_state, double p, int64_t micro, int64_t site,
                                const OptTensor& sids, const OptTensor& cu) {
  DeviceGuard guard(qkv.device());
  chk16(qkv, "qkv");
  TORCH_CHECK(qkv.is_contiguous() && (cu.has_value() || qkv.size(0) == B * S) && qkv.size(1) == 3 * A * 64,
              "qkv must be [B*S, 3*A*64]");
  Tensor ctx = at::empty({qkv.size(0), A * 64}, qkv.options());
  Tensor lse = at::empty({B, A, S}, qkv.options().dtype(at::kFloat));
  PdtRng rng{nullptr, 0, 0};
  if (rng_state.has_value()) rng = make_rng(*rng_state, micro, site, sids, S, B);
  check(pdt_attn_fwd(dt_code(qkv), qkv.data_ptr(), mask.data_ptr<int32_t>(), kv_len.data_ptr<int32_t>(),
                     cu.has_value() ? cu->data_ptr<int32_t>() : nullptr, ctx.data_ptr(),
                     lse.data_ptr<float>(), (int)B, (int)S, (int)A, keep_scale(p), thr16(p), rng, cur_stream()), "attn_fwd");
  return {ctx, lse};
}
Tensor op_attn_bwd(const Tensor& qkv, const Tensor& mask, const Tensor& kv_len, const Tensor& ctx, const Tensor& dctx,
                   const Tensor& lse, int64_t B, int64_t S, int64_t A, const c10::optional<Tensor>& rng_state, double p,
                   int64_t micro, int64_t site, c10::optional<Tensor> dbias, const OptTensor& sids, const OptTensor& cu) {
  DeviceGuard guard(qkv.device());
  Tensor dqkv = at::empty_like(qkv);
  Tensor delta = at::empty_like(lse);
  Tensor dc = dctx.contiguous();
  PdtRng rng{nullptr, 0, 0};
  if (rng_state.has_value()) rng = make_rng(*rng_state, micro, site, sids, S, B);
  // `dbias` (fp32 [3H]): the column sums of dqkv are added to it (short-sequence kernel only)
  const int64_t H3 = qkv.size(1);
  Tensor part;
  const int db_rows = pdt_attn_bwd_dbias_rows((int)B, (int)S);
  if (dbias.has_value()) { chkf32(*dbias, "dbias"); part = at::empty({(int64_t)db_rows, H3}, lse.options()); }
  check(pdt_attn_bwd(dt_code(qkv), qkv.data_ptr(), mask.data_ptr<int32_t>(), kv_len.data_ptr<int32_t>(),
                     cu.has_value() ? cu->data_ptr<int32_t>() : nullptr, ctx.data_ptr(),
                     dc.data_ptr(), lse.data_ptr<float>(), delta.data_ptr<float>(), dqkv.data_ptr(),
                     dbias.has_value() ? part.data_ptr<float>() : nullptr, (int)B, (int)S, (int)A, keep_scale(p),
                     thr16(p), rng, cur_stream()), "attn_bwd");
  if (dbias.has_value())
    check(pdt_colsum_finish(part.data_ptr<float>(), db_rows, (int)H3, 1, dbias->data_ptr<float>(), nullptr, nullptr, nullptr, 1,
                            cur_stream()), "colsum_finish");
  return dqkv;
}

}  // namespace

void bind_rccl_comm(py::module_& m);  // rccl_comm.cpp
void bind_reducer(py::module_& m);    // reducer.cpp
void bind_wordpiece(py::module_& m);  // wordpiece.cpp

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "gfx950 kernels + native runtime of pytorch_distributed_training_amd";
  // (the trailing `sample_ids` arguments: optional int32 [B] global sample ids for sample-keyed dropout, see PdtRng)
  // The GIL is released while a call issues its launches (25-30 HIP calls for a layer's backward): a second Python
  // thread can enqueue the next micro-batch's forward on its own stream meanwhile (Engine.accumulate) - short
  // micro-batches are bound by the rate at which ONE host thread can launch kernels.
  using nogil = py::call_guard<py::gil_scoped_release>;
  py::class_<LayerPosition, LayerPositionPtr>(m, "LayerPosition", "position options of an encoder layer's attention")
      .def(py::init<>())
      .def_readwrite("table", &LayerPosition::table)
      .def_readwrite("wq", &LayerPosition::wq)
      .def_readwrite("wk", &LayerPosition::wk)
      .def_readwrite("cos", &LayerPosition::cos)
      .def_readwrite("sin", &LayerPosition::sin)
      .def_readwrite("max_distance", &LayerPosition::max_distance)
      .def_readwrite("steps", &LayerPosition::steps)
      .def_readwrite("eps", &LayerPosition::eps);
  m.def("layer_forward", &layer_forward, nogil());
  m.def("layer_backward", &layer_backward, nogil());
  m.def("stack_forward", &stack_forward, nogil());
  m.def("stack_backward", &stack_backward, nogil());
  m.def("embed_forward", &embed_forward, nogil());
  m.def("embed_backward", &embed_backward, nogil());
  m.def("dense_tanh_forward", &dense_tanh_forward, nogil());
  m.def("dense_backward", &dense_backward, nogil());
  m.def("head_forward", &head_forward, nogil());
  m.def("head_backward", &head_backward, nogil());
  m.def("dropout16", &dropout16);
  m.def("rel_mask_bits", &rel_mask_bits);
  m.def("rel_attn_forward", &rel_attn_forward, nogil());
  m.def("rel_attn_backward", &rel_attn_backward, nogil());
  m.def("relative_attention", &relative_attention, nogil());
  m.def("qk_norm_rope", &qk_norm_rope, nogil());
  m.def("qk_rope_forward", &qk_rope_forward, nogil());
  m.def("qk_rope_backward", &qk_rope_backward, nogil());
  m.def("adamw_step", &adamw_step);
  m.def("grad_check", &grad_check);
  m.def("scaler_update", &scaler_update);
  m.def("cast_to_16", &cast_to_16);
  m.def("op_gemm", &op_gemm, py::arg("layout"), py::arg("A"), py::arg("B"), py::arg("epi"), py::arg("bias"),
        py::arg("res"), py::arg("aux"), py::arg("rng_state"), py::arg("drop_p"), py::arg("micro"), py::arg("site"),
        py::arg("tile"), py::arg("colsum") = py::none(), py::arg("sample_ids") = py::none(), py::arg("seq") = 1);
  m.def("op_gemm_tn", &op_gemm_tn);
  m.def("gemm_splits", [](const std::string& layout, const Tensor& A, const Tensor& B) {
    PdtGemm g{};
    g.M = (int)A.size(0); g.K = (int)A.size(1); g.N = (int)(layout == "nt" ? B.size(0) : B.size(1));
    return pdt_gemm_splits(layout == "nt" ? PDT_GEMM_NT : PDT_GEMM_NN, -1, &g);
  }, "K slices the dispatcher uses for a forward (nt) / dgrad (nn) GEMM of these operands (1 = one kernel)");
  m.def("op_layernorm_fwd", &op_layernorm_fwd);
  m.def("op_layernorm_bwd", &op_layernorm_bwd, py::arg("dy"), py::arg("x"), py::arg("stats"), py::arg("gamma"),
        py::arg("rng_state"), py::arg("drop_p"), py::arg("micro"), py::arg("site"), py::arg("sample_ids") = py::none(),
        py::arg("seq") = 1);
  m.def("op_attn_fwd", &op_attn_fwd, py::arg("qkv"), py::arg("mask"), py::arg("kv_len"), py::arg("B"), py::arg("S"), py::arg("A"),
        py::arg("rng_state"), py::arg("p"), py::arg("micro"), py::arg("site"), py::arg("sample_ids") = py::none(),
        py::arg("cu_seqlens") = py::none());
  m.def("op_attn_bwd", &op_attn_bwd, py::arg("qkv"), py::arg("mask"), py::arg("kv_len"), py::arg("ctx"), py::arg("dctx"),
        py::arg("lse"), py::arg("B"), py::arg("S"), py::arg("A"), py::arg("rng_state"), py::arg("p"), py::arg("micro"),
        py::arg("site"), py::arg("dbias") = py::none(), py::arg("sample_ids") = py::none(), py::arg("cu_seqlens") = py::none());
  m.def("set_wgrad_defer", [](bool on) { g_wgrad_defer = on; },
        "queue a layer's weight-gradient GEMMs behind one fork and skip the per-layer join (call wgrad_join after backward)");
  m.def("wgrad_join", [] { WgradLane::join_deferred(); },
        "current stream waits for the deferred weight-gradient GEMMs issued from it; releases the tensors kept for them");
  m.def("set_wgrad_side_stream", [](int64_t mode) { g_wgrad_mode = (int)mode; },
        "weight-gradient GEMMs of layer_backward on a second HIP stream: 0 never, 1 up to 12288 tokens (default), 2 always");
  m.def("set_gemm_persistent", [](int64_t mode) { pdt_gemm_set_persist_mode((int)mode); },
        "persistent launches of the ping-pong GEMM: 0 never, 1 from 4 tiles per workgroup (default), 2 from 2");
  m.def("gemm_persistent_mode", [] { return pdt_gemm_persist_mode(); });
  m.def("set_gemm_split_k", [](bool on) { pdt_gemm_set_split_mode(on ? 1 : 0); },
        "K split of forward / dgrad GEMMs with few output tiles: on (default) for latency-bound lone micro-batches, off "
        "while two micro-batches overlap on two streams");
  m.def("gemm_split_k", [] { return pdt_gemm_split_mode() != 0; });
  m.def("set_debug_sync", [](bool on) { g_debug_sync = on; },
        "drain the device after every native launch and report a fault at the op that caused it");
  m.def("debug_sync_count", [] { return g_debug_sync_count; });
  m.def("attn_bwd_fuses_dbias", [](int64_t S) { return pdt_attn_bwd_fuses_dbias((int)S) != 0; });
  bind_rccl_comm(m);  // (before the reducer: its constructor signature names RcclComm)
  bind_reducer(m);
  bind_wordpiece(m);
}
