// PyTorch-ROCm operator registration for the fp64_emu ops.  The schemas are
// the reference's (torch-ext/torch_binding.cpp:7-12) and the argument checks
// raise its TORCH_CHECK messages (fp64_emu_cuda/fp64_emu.cu:1586-1600,
// 1616-1628, 1640-1654, 1668-1682, 1692-1693).  Each op validates, takes its
// scratch from the caching allocator on the current stream and calls the C
// ABI of include/fp64emu.h; nothing here computes.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include <algorithm>
#include <optional>
#include <utility>
#include <vector>

#include "fp64emu.h"

namespace {

constexpr int64_t kMaxKSingle = 131071;
constexpr int64_t kMaxKDeep = (int64_t)128 * 65536;   // the deep bound (mm, bmm)

void check_status(int st) { TORCH_CHECK(st == FP64EMU_OK, fp64emu_last_error()); }

std::vector<int32_t> primes_vec(const at::Tensor& primes_cpu) {
  const at::Tensor pc = primes_cpu.to(at::kCPU, at::kInt).contiguous();
  const int32_t* p = pc.data_ptr<int32_t>();
  return std::vector<int32_t>(p, p + pc.numel());
}

at::Tensor workspace(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// The full workspace when the caching allocator can provide it; otherwise the
// staged form's, where that is smaller (the planes of a whole-K product are
// several times its segmented ones); otherwise the largest of half, a quarter,
// ... of that down to the minimum the library accepts (it then runs the rows
// of A in as few chunks as fit: batch-1 calls with K <= 131071).
template <typename Size>
at::Tensor workspace_fit(const at::Tensor& like, size_t full, const Size& size) {
  try {
    return workspace(like, full);
  } catch (const c10::OutOfMemoryError&) {
  }
  const size_t staged = size(fp64emu_workspace_size), minimum = size(fp64emu_workspace_size_min);
  for (size_t want = staged < full ? staged : full / 2; want > minimum; want /= 2) {
    try {
      return workspace(like, want);
    } catch (const c10::OutOfMemoryError&) {
    }
  }
  return workspace(like, minimum);
}

fp64emu_stream_t current_stream(const at::Tensor& t) {
  return reinterpret_cast<fp64emu_stream_t>(
      c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_common(const at::Tensor& A, const at::Tensor& B, const char* dtype_msg,
                  const at::Tensor& primes_cpu, int64_t bits) {
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.scalar_type() == at::kDouble &&
                  B.scalar_type() == at::kDouble,
              dtype_msg);
  TORCH_CHECK(A.device() == B.device(), "A and B must be on the same device");
  TORCH_CHECK(primes_cpu.numel() <= FP64EMU_MAXP, "too many primes");
  TORCH_CHECK(primes_cpu.numel() >= 1, "nprimes must be >= 1");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
}

void check_out(const at::Tensor& out, const at::Tensor& A, at::IntArrayRef sizes,
               const char* msg) {
  TORCH_CHECK(out.scalar_type() == at::kDouble && out.sizes() == sizes && out.is_contiguous(),
              msg);
  TORCH_CHECK(out.device() == A.device(), "out must be on the device of A");
}

// The product of checked operands (A as [batch, M, K]) into out.
void product(at::Tensor& out, const at::Tensor& A, const at::Tensor& B, int64_t batch, int64_t M,
             int64_t N, int64_t K, bool b_kn, const at::Tensor& primes_cpu, bool exact, int64_t bits,
             bool use_corr) {
  const c10::DeviceGuard guard(A.device());
  const std::vector<int32_t> pv = primes_vec(primes_cpu);
  fp64emu_product_t p;
  p.out = out.data_ptr<double>();
  p.A = A.data_ptr<double>();
  p.B = B.data_ptr<double>();
  p.batch = batch; p.M = M; p.N = N; p.K = K;
  p.b_kn = b_kn;
  p.primes = pv.data();
  p.nprimes = (int)pv.size();
  p.exact = exact;
  p.bits = bits;
  p.use_corr = use_corr;
  at::Tensor ws = workspace_fit(A, fp64emu_product_workspace(&p), [&](auto workspace_size) {
    return workspace_size(batch, M, N, K, p.nprimes, use_corr);
  });
  check_status(fp64emu_product(&p, ws.data_ptr(), (size_t)ws.numel(), current_stream(A)));
}

}  // namespace

int64_t fp64_emu_maxp() { return fp64emu_maxp(); }

// out[m,n] = A[m,k] @ B[n,k]^T.   fp64_emu_cuda/fp64_emu.cu:1583-1608
void fp64_emu_mm(at::Tensor& out, const at::Tensor& A, const at::Tensor& B,
                 const at::Tensor& primes_cpu, const at::Tensor& inv_cpu,
                 const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu; (void)mu_cpu;
  check_common(A, B, "A,B must be f64 CUDA", primes_cpu, bits);
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && A.is_contiguous() && B.is_contiguous(), "2D contig");
  const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
  TORCH_CHECK(B.size(1) == K, "expect B as [N, K]");
  check_out(out, A, {M, N}, "out f64 [M,N]");
  // Past one launch's 131071, whole or K-segmented: to 128 segments of 65536.
  TORCH_CHECK(K <= kMaxKDeep, "K bound: 128 segments of 65536");
  product(out, A, B, 1, M, N, K, false, primes_cpu, exact, bits, use_corr);
}

// out[m,n] = A[m,k] @ Bt[k,n], Bt in its [K, N] layout.
// fp64_emu_cuda/fp64_emu.cu:1613-1632
void fp64_emu_mm_nt(at::Tensor& out, const at::Tensor& A, const at::Tensor& Bt,
                    const at::Tensor& primes_cpu, const at::Tensor& inv_cpu,
                    const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu; (void)mu_cpu;
  check_common(A, Bt, "A,Bt must be f64 CUDA", primes_cpu, bits);
  TORCH_CHECK(A.dim() == 2 && Bt.dim() == 2 && A.is_contiguous() && Bt.is_contiguous(),
              "2D contig");
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(1);
  TORCH_CHECK(Bt.size(0) == K, "expect Bt as [K, N]");
  check_out(out, A, {M, N}, "out f64 [M,N]");
  TORCH_CHECK(K <= kMaxKSingle, "K bound for int32 modular GEMM");
  product(out, A, Bt, 1, M, N, K, true, primes_cpu, exact, bits, use_corr);
}

// out[b,m,n] = A[b,m,k] @ B[b,n,k]^T.   fp64_emu_cuda/fp64_emu.cu:1637-1662
void fp64_emu_bmm(at::Tensor& out, const at::Tensor& A, const at::Tensor& B,
                  const at::Tensor& primes_cpu, const at::Tensor& inv_cpu,
                  const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu; (void)mu_cpu;
  check_common(A, B, "A,B must be f64 CUDA", primes_cpu, bits);
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.is_contiguous() && B.is_contiguous(), "3D contig");
  const int64_t batch = A.size(0), M = A.size(1), K = A.size(2), N = B.size(1);
  TORCH_CHECK(B.size(0) == batch && B.size(2) == K, "expect B as [batch, N, K]");
  check_out(out, A, {batch, M, N}, "out f64 [batch,M,N]");
  TORCH_CHECK(K <= kMaxKDeep, "K bound: 128 segments of 65536");
  product(out, A, B, batch, M, N, K, false, primes_cpu, exact, bits, use_corr);
}

// out[b,m,n] = A[b,m,k] @ Bt[b,k,n].   fp64_emu_cuda/fp64_emu.cu:1665-1686
void fp64_emu_bmm_nt(at::Tensor& out, const at::Tensor& A, const at::Tensor& Bt,
                     const at::Tensor& primes_cpu, const at::Tensor& inv_cpu,
                     const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu; (void)mu_cpu;
  check_common(A, Bt, "A,Bt must be f64 CUDA", primes_cpu, bits);
  TORCH_CHECK(A.dim() == 3 && Bt.dim() == 3 && A.is_contiguous() && Bt.is_contiguous(),
              "3D contig");
  const int64_t batch = A.size(0), M = A.size(1), K = A.size(2), N = Bt.size(2);
  TORCH_CHECK(Bt.size(0) == batch && Bt.size(1) == K, "expect Bt as [batch, K, N]");
  check_out(out, A, {batch, M, N}, "out f64 [batch,M,N]");
  TORCH_CHECK(K <= kMaxKSingle, "K bound for int32 modular GEMM");
  product(out, A, Bt, batch, M, N, K, true, primes_cpu, exact, bits, use_corr);
}

// mm with phase times [scale+extract, gemms, marker, reconstruct] in ms.
// fp64_emu_cuda/fp64_emu.cu:1688-1704 (plus the dtype/shape checks it lacks).
void fp64_emu_mm_timed(at::Tensor& out, at::Tensor& times, const at::Tensor& A,
                       const at::Tensor& B, const at::Tensor& primes_cpu,
                       const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact,
                       int64_t bits, bool use_corr) {
  (void)inv_cpu; (void)mu_cpu;
  check_common(A, B, "A,B must be f64 CUDA", primes_cpu, bits);
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && A.is_contiguous() && B.is_contiguous(), "2D contig");
  const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
  TORCH_CHECK(B.size(1) == K, "expect B as [N, K]");
  check_out(out, A, {M, N}, "out f64 [M,N]");
  TORCH_CHECK(K <= kMaxKSingle, "K bound for int32 modular GEMM");
  TORCH_CHECK(times.device().is_cpu() && times.scalar_type() == at::kFloat &&
                  times.numel() >= 4 && times.is_contiguous(),
              "times must be a CPU float32 tensor of 4");
  const c10::DeviceGuard guard(A.device());
  const std::vector<int32_t> pv = primes_vec(primes_cpu);
  const int P = (int)pv.size();
  at::Tensor ws = workspace(A, fp64emu_workspace_size(1, M, N, K, P, use_corr));
  check_status(fp64emu_mm_timed(out.data_ptr<double>(), times.data_ptr<float>(),
                                A.data_ptr<double>(), B.data_ptr<double>(), M, N, K, pv.data(),
                                nullptr, nullptr, P, exact, bits, use_corr, ws.data_ptr(),
                                (size_t)ws.numel(), current_stream(A)));
}

// ---- Operands in 8-bit floating point (include/fp64emu.h, fp64emu_f8_t) ----
namespace {

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FP64EMU_F32;
    case at::kBFloat16: return FP64EMU_BF16;
    case at::kHalf: return FP64EMU_F16;
    default: TORCH_CHECK(false, "expect float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

// t where its rows are contiguous and do not overlap (those of an expanded tensor do),
// else a contiguous copy.
at::Tensor in_rows(const at::Tensor& t) {
  const int64_t d = t.dim(), w = t.size(d - 1);
  const bool fine = (w <= 1 || t.stride(d - 1) == 1) && (t.size(d - 2) <= 1 || t.stride(d - 2) >= w);
  return fine ? t : t.contiguous();
}

// q [(batch,) rows, depth] and its scales [(batch,) rows or tile rows, blocks].
fp64emu_f8_t f8_of(const at::Tensor& q, const at::Tensor& s, const char* what) {
  fp64emu_f8_t f{};
  const auto type = q.scalar_type();
  TORCH_CHECK(type == at::kFloat8_e4m3fn || type == at::kFloat8_e5m2, what,
              ": codes are float8_e4m3fn or float8_e5m2, got ", type);
  TORCH_CHECK(s.scalar_type() == at::kFloat, what, ": scales are float32");
  TORCH_CHECK(q.is_cuda() && s.is_cuda() && q.device() == s.device(), what,
              ": codes and scales must be on one GPU");
  const int64_t d = q.dim();
  TORCH_CHECK((d == 2 || d == 3) && s.dim() == d, what, ": codes and scales are both 2-D or both 3-D");
  const int64_t rows = q.size(d - 2), depth = q.size(d - 1);
  TORCH_CHECK(d == 2 || s.size(0) == q.size(0), what, ": batch of codes and scales");
  TORCH_CHECK(s.size(d - 1) == (depth + 127) / 128, what, ": expect one scale per 128 of K, ",
              (depth + 127) / 128, ", got ", s.size(d - 1));
  TORCH_CHECK(s.size(d - 2) == rows || s.size(d - 2) == (rows + 127) / 128, what,
              ": expect scales by rows or by tiles of 128 rows");
  f.q = static_cast<uint8_t*>(q.data_ptr());
  f.s = s.data_ptr<float>();
  f.ld = rows > 1 ? q.stride(d - 2) : std::max<int64_t>(depth, (depth + 15) / 16 * 16);
  TORCH_CHECK(f.ld >= depth, what, ": rows of codes overlap");
  f.stride = d == 3 && q.size(0) > 1 ? q.stride(0) : 0;
  f.s_row = s.stride(d - 2);
  f.s_block = s.stride(d - 1);
  f.s_stride = d == 3 ? s.stride(0) : 0;
  f.fmt = type == at::kFloat8_e4m3fn ? FP64EMU_E4M3 : FP64EMU_E5M2;
  f.tiles = s.size(d - 2) != rows;
  return f;
}

void check_rows(const at::Tensor& t, const char* what) {
  const int64_t d = t.dim();
  TORCH_CHECK(t.is_cuda(), what, " must be on a GPU");
  TORCH_CHECK(t.size(d - 1) <= 1 || t.stride(d - 1) == 1, what, " must be contiguous along its rows");
}

int64_t row_stride(const at::Tensor& t) {
  const int64_t d = t.dim(), w = t.size(d - 1);
  const int64_t ld = t.size(d - 2) > 1 ? t.stride(d - 2) : (w + 7) / 8 * 8;
  TORCH_CHECK(ld >= w, "rows overlap");
  return ld;
}

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// A new quantised matrix [(batch,) rows, depth]: codes in rows of a multiple of 16
// bytes, which the product copies fastest, scales stored block by block, in the
// order it reads them.
struct NewF8 {
  at::Tensor q, s;
  fp64emu_f8_t f{};
  NewF8(const at::Tensor& like, const int64_t* batch, int64_t rows, int64_t depth, int64_t scale_rows,
        int64_t blocks, at::ScalarType fmt, bool tiles) {
    const int64_t ld = (depth + 15) / 16 * 16, n = batch ? *batch : 1;
    const at::TensorOptions on = like.options();
    if (batch) {
      q = at::empty({n, rows, ld}, on.dtype(fmt));
      s = at::empty_strided({n, scale_rows, blocks}, {scale_rows * blocks, 1, scale_rows}, on.dtype(at::kFloat));
    } else {
      q = at::empty({rows, ld}, on.dtype(fmt));
      s = at::empty_strided({scale_rows, blocks}, {1, scale_rows}, on.dtype(at::kFloat));
    }
    if (ld != depth) q = q.narrow(-1, 0, depth);
    f.q = static_cast<uint8_t*>(q.data_ptr());
    f.s = s.data_ptr<float>();
    f.ld = ld;
    f.stride = rows * ld;
    f.s_row = 1;
    f.s_block = scale_rows;
    f.s_stride = scale_rows * blocks;
    f.fmt = fmt == at::kFloat8_e4m3fn ? FP64EMU_E4M3 : FP64EMU_E5M2;
    f.tiles = tiles;
  }
};

fp64emu_f8_t kept_of(const at::Tensor& like, const at::Tensor& hq, const at::Tensor& hs, int64_t M, int64_t F) {
  TORCH_CHECK(hq.sizes() == at::IntArrayRef({M, 2 * F}) && hq.scalar_type() == at::kFloat8_e4m3fn,
              "hq float8_e4m3fn [M, 2 F]");
  TORCH_CHECK(hs.sizes() == at::IntArrayRef({M, 2 * blocks_of(F)}) && hs.scalar_type() == at::kFloat,
              "hs float32 [M, 2 ceil(F / 128)]");
  TORCH_CHECK(hq.device() == like.device() && hs.device() == like.device(),
              "dy, hq and hs must be on the same device");
  check_rows(hq, "hq");
  fp64emu_f8_t f{};
  f.q = static_cast<uint8_t*>(hq.data_ptr());
  f.s = hs.data_ptr<float>();
  f.ld = row_stride(hq);
  f.s_row = hs.stride(0);
  f.s_block = hs.stride(1);
  return f;
}

constexpr int64_t kPlain = 0, kRows = 1, kBoth = 2;    // what form an activation's result takes

void product_f8(const at::Tensor& out, const at::Tensor& A, const at::Tensor& sA, const at::Tensor& B,
                const at::Tensor& sB, bool accumulate) {
  TORCH_CHECK(A.dim() >= 2 && B.dim() >= 2 && out.dim() >= 2, "A, B and out are all 2-D or all 3-D");
  const at::Tensor qa = in_rows(A), qb = in_rows(B);
  fp64emu_mm_f8_t p{};
  p.A = f8_of(qa, sA, "A");
  p.B = f8_of(qb, sB, "B");
  const int64_t d = A.dim();
  TORCH_CHECK(B.dim() == d && out.dim() == d, "A, B and out are all 2-D or all 3-D");
  TORCH_CHECK(A.device() == B.device() && A.device() == out.device(),
              "A, B and out must be on the same device");
  p.batch = d == 3 ? A.size(0) : 1;
  p.M = A.size(d - 2);
  p.K = A.size(d - 1);
  p.N = B.size(d - 2);
  TORCH_CHECK(B.size(d - 1) == p.K && (d == 2 || B.size(0) == p.batch),
              d == 2 ? "expect B as [N, K]" : "expect B as [batch, N, K]");
  TORCH_CHECK(sA.size(d - 2) == p.M, "A's scales are by rows");
  p.A.tiles = 0;
  TORCH_CHECK(out.size(d - 2) == p.M && out.size(d - 1) == p.N && (d == 2 || out.size(0) == p.batch),
              "out [M, N] of the product");
  check_rows(out, "out");
  p.out = out.data_ptr();
  p.dtype = dtype_of(out);
  p.ldo = row_stride(out);
  p.stride_o = d == 3 && p.batch > 1 ? out.stride(0) : 0;
  p.accumulate = accumulate;
  const c10::DeviceGuard guard(A.device());
  const size_t bytes = fp64emu_mm_f8_workspace(&p);
  at::Tensor ws;
  if (bytes) ws = workspace(A, bytes);
  check_status(fp64emu_mm_f8(&p, bytes ? ws.data_ptr() : nullptr, bytes, current_stream(A)));
}

}  // namespace

// x [(batch,) M, K] into (q, s) by rows, (qt, st) by columns laid transposed, or
// both; `tiles`: one scale for 128 x 128.
std::vector<at::Tensor> fp64_emu_quant_f8(const at::Tensor& x, bool rows, bool cols, bool tiles,
                                          at::ScalarType fmt) {
  const int64_t d = x.dim();
  TORCH_CHECK(d == 2 || d == 3, "expect x as [M, K] or [batch, M, K]");
  TORCH_CHECK(fmt == at::kFloat8_e4m3fn || fmt == at::kFloat8_e5m2, "fmt must be float8_e4m3fn or float8_e5m2");
  const at::Tensor v = in_rows(x);
  check_rows(v, "x");
  const int dtype = dtype_of(v);
  const int64_t batch = d == 3 ? v.size(0) : 1, M = v.size(d - 2), K = v.size(d - 1);
  const int64_t MB = blocks_of(M), KB = blocks_of(K), *b = d == 3 ? &batch : nullptr;
  const c10::DeviceGuard guard(v.device());
  std::optional<NewF8> r, c;
  std::vector<at::Tensor> out;
  if (rows) {
    r.emplace(v, b, M, K, tiles ? MB : M, KB, fmt, tiles);
    out.insert(out.end(), {r->q, r->s});
  }
  if (cols) {
    c.emplace(v, b, K, M, tiles ? KB : K, MB, fmt, tiles);
    out.insert(out.end(), {c->q, c->s});
  }
  check_status(fp64emu_quant_f8(v.data_ptr(), dtype, batch, M, K, row_stride(v),
                                batch > 1 ? v.stride(0) : 0, r ? &r->f : nullptr, c ? &c->f : nullptr,
                                current_stream(v)));
  return out;
}

// sum_k A[(b,) m, k] B[(b,) n, k] as a new tensor of `dtype`.
at::Tensor fp64_emu_mm_f8(const at::Tensor& A, const at::Tensor& sA, const at::Tensor& B, const at::Tensor& sB,
                          at::ScalarType dtype) {
  const int64_t d = A.dim();
  TORCH_CHECK((d == 2 || d == 3) && B.dim() == d, "A, B and out are all 2-D or all 3-D");
  const at::TensorOptions on = A.options().dtype(dtype);
  const at::Tensor out = d == 3 ? at::empty({A.size(0), A.size(1), B.size(1)}, on)
                                : at::empty({A.size(0), B.size(0)}, on);
  product_f8(out, A, sA, B, sB, false);
  return out;
}

// The same into out, or added to it.
void fp64_emu_mm_f8_out(at::Tensor& out, const at::Tensor& A, const at::Tensor& sA, const at::Tensor& B,
                        const at::Tensor& sB, bool accumulate) {
  at::assert_no_internal_overlap(out);
  product_f8(out, A, sA, B, sB, accumulate);
}

// y = silu(g) u of h = [g | u]: y, or its (q, s), or (q, s, qt, st); then, with
// keep, (hq, hs).
std::vector<at::Tensor> fp64_emu_swiglu_f8(const at::Tensor& h, int64_t quant, bool keep) {
  TORCH_CHECK(h.dim() == 2 && h.size(1) % 2 == 0, "expect h as [M, 2 F]");
  TORCH_CHECK(quant >= kPlain && quant <= kBoth, "quant: 0 plain, 1 rows, 2 both");
  const at::Tensor v = in_rows(h);
  check_rows(v, "h");
  const int dtype = dtype_of(v);
  const int64_t M = v.size(0), F = v.size(1) / 2, FB = blocks_of(F);
  const c10::DeviceGuard guard(v.device());
  std::optional<NewF8> r, c, k;
  at::Tensor y;
  std::vector<at::Tensor> out;
  if (quant == kPlain) {
    y = at::empty({M, F}, v.options());
    out.push_back(y);
  } else {
    r.emplace(v, nullptr, M, F, M, FB, at::kFloat8_e4m3fn, false);
    out.insert(out.end(), {r->q, r->s});
  }
  if (quant == kBoth) {
    c.emplace(v, nullptr, F, M, F, blocks_of(M), at::kFloat8_e4m3fn, false);
    out.insert(out.end(), {c->q, c->s});
  }
  if (keep) {
    k.emplace(v, nullptr, M, 2 * F, M, 2 * FB, at::kFloat8_e4m3fn, false);
    out.insert(out.end(), {k->q, k->s});
  }
  check_status(fp64emu_swiglu_f8(v.data_ptr(), dtype, M, F, row_stride(v), y.defined() ? y.data_ptr() : nullptr, F,
                                 k ? &k->f : nullptr, r ? &r->f : nullptr, c ? &c->f : nullptr,
                                 current_stream(v)));
  return out;
}

// The gradient of fp64_emu_swiglu_f8 from what it kept: dh, or its (q, s), or (q, s, qt, st).
std::vector<at::Tensor> fp64_emu_swiglu_f8_backward(const at::Tensor& dy, const at::Tensor& hq,
                                                    const at::Tensor& hs, int64_t quant) {
  TORCH_CHECK(dy.dim() == 2, "expect dy as [M, F]");
  TORCH_CHECK(quant >= kPlain && quant <= kBoth, "quant: 0 plain, 1 rows, 2 both");
  const at::Tensor v = in_rows(dy);
  check_rows(v, "dy");
  const int dtype = dtype_of(v);
  const int64_t M = v.size(0), F = v.size(1);
  const at::Tensor codes = in_rows(hq);
  const fp64emu_f8_t keep = kept_of(v, codes, hs, M, F);
  const c10::DeviceGuard guard(v.device());
  // Blocks of the whole 2 F that straddle the halves are quantised in a pass of
  // their own, from float32 so that nothing is rounded twice.
  const bool straddle = quant != kPlain && F % 128 != 0;
  if (quant == kPlain || straddle) {
    const at::Tensor dh = at::empty({M, 2 * F}, straddle ? v.options().dtype(at::kFloat) : v.options());
    check_status(fp64emu_swiglu_f8_backward(v.data_ptr(), dtype, M, F, row_stride(v), &keep, dh.data_ptr(),
                                            dtype_of(dh), 2 * F, nullptr, nullptr, current_stream(v)));
    if (!straddle) return {dh};
    return fp64_emu_quant_f8(dh, true, quant == kBoth, false, at::kFloat8_e4m3fn);
  }
  std::optional<NewF8> r, c;
  r.emplace(v, nullptr, M, 2 * F, M, blocks_of(2 * F), at::kFloat8_e4m3fn, false);
  std::vector<at::Tensor> out{r->q, r->s};
  if (quant == kBoth) {
    c.emplace(v, nullptr, 2 * F, M, 2 * F, blocks_of(M), at::kFloat8_e4m3fn, false);
    out.insert(out.end(), {c->q, c->s});
  }
  check_status(fp64emu_swiglu_f8_backward(v.data_ptr(), dtype, M, F, row_stride(v), &keep, nullptr, dtype, 0,
                                          &r->f, c ? &c->f : nullptr, current_stream(v)));
  return out;
}

TORCH_LIBRARY(fp64_emu, ops) {
  ops.def("fp64_emu_maxp() -> int", &fp64_emu_maxp);
  ops.def("fp64_emu_mm(Tensor! out, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def("fp64_emu_bmm(Tensor! out, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def("fp64_emu_mm_nt(Tensor! out, Tensor A, Tensor Bt, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def("fp64_emu_bmm_nt(Tensor! out, Tensor A, Tensor Bt, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def("fp64_emu_mm_timed(Tensor! out, Tensor! times, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def("fp64_emu_quant_f8(Tensor x, bool rows, bool cols, bool tiles, ScalarType fmt) -> Tensor[]");
  ops.def("fp64_emu_mm_f8(Tensor A, Tensor sA, Tensor B, Tensor sB, ScalarType dtype) -> Tensor");
  ops.def("fp64_emu_mm_f8_out(Tensor(a!) out, Tensor A, Tensor sA, Tensor B, Tensor sB, bool accumulate) -> ()");
  ops.def("fp64_emu_swiglu_f8(Tensor h, int quant, bool keep) -> Tensor[]");
  ops.def("fp64_emu_swiglu_f8_backward(Tensor dy, Tensor hq, Tensor hs, int quant) -> Tensor[]");
}

// PyTorch-ROCm keeps the CUDA dispatch key for HIP devices.
TORCH_LIBRARY_IMPL(fp64_emu, CUDA, ops) {
  ops.impl("fp64_emu_mm", &fp64_emu_mm);
  ops.impl("fp64_emu_bmm", &fp64_emu_bmm);
  ops.impl("fp64_emu_mm_nt", &fp64_emu_mm_nt);
  ops.impl("fp64_emu_bmm_nt", &fp64_emu_bmm_nt);
  ops.impl("fp64_emu_mm_timed", &fp64_emu_mm_timed);
  ops.impl("fp64_emu_quant_f8", &fp64_emu_quant_f8);
  ops.impl("fp64_emu_mm_f8", &fp64_emu_mm_f8);
  ops.impl("fp64_emu_mm_f8_out", &fp64_emu_mm_f8_out);
  ops.impl("fp64_emu_swiglu_f8", &fp64_emu_swiglu_f8);
  ops.impl("fp64_emu_swiglu_f8_backward", &fp64_emu_swiglu_f8_backward);
}

// None of the 8-bit ops has a derivative: a result that would need one raises in the
// backward pass, an `out` that would need one at once.
namespace {

using MmOut = void(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, bool);

const c10::TypedOperatorHandle<MmOut>& mm_out_handle() {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("fp64_emu::fp64_emu_mm_f8_out", "").typed<MmOut>();
  return op;
}

void mm_f8_out_autograd(c10::DispatchKeySet keys, at::Tensor& out, const at::Tensor& A, const at::Tensor& sA,
                        const at::Tensor& B, const at::Tensor& sB, bool accumulate) {
  if (at::GradMode::is_enabled())
    for (const at::Tensor* t : {(const at::Tensor*)&out, &A, &sA, &B, &sB})
      TORCH_CHECK(!t->requires_grad(), "the derivative for a product into out is not implemented, ",
                  "but one of its arguments requires a gradient");
  mm_out_handle().redispatch(keys & c10::after_autograd_keyset, out, A, sA, B, sB, accumulate);
}

void mm_f8_out_written(c10::DispatchKeySet keys, at::Tensor& out, const at::Tensor& A, const at::Tensor& sA,
                       const at::Tensor& B, const at::Tensor& sB, bool accumulate) {
  mm_out_handle().redispatch(keys & c10::after_ADInplaceOrView_keyset, out, A, sA, B, sB, accumulate);
  out.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

TORCH_LIBRARY_IMPL(fp64_emu, Autograd, ops) {
  for (const char* name : {"fp64_emu_quant_f8", "fp64_emu_mm_f8", "fp64_emu_swiglu_f8", "fp64_emu_swiglu_f8_backward"})
    ops.impl(name, torch::autograd::autogradNotImplementedFallback());
  ops.impl("fp64_emu_mm_f8_out", &mm_f8_out_autograd);
}

TORCH_LIBRARY_IMPL(fp64_emu, ADInplaceOrView, ops) { ops.impl("fp64_emu_mm_f8_out", &mm_f8_out_written); }
