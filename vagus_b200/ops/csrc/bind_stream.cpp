// Bindings of the long-context streaming operators: rotary positions
// (rotary.cu), the 4-bit key / value cache and attention over it (kv4.cu) and
// the verification of drafted tokens (verify.cu).  Every op runs on its
// tensors' device, on that device's current stream.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "kernels.h"

int* vagus_device_error_ptr();   // bindings.cpp

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "vagus_b200 kernel '", what, "' rejected the problem or failed to launch (code ", rc, ")");
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

int type_of(const Tensor& t, const char* what) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kFloat || s == at::kHalf || s == at::kBFloat16, what, ": fp32, fp16 or bf16");
  return s == at::kFloat ? 0 : s == at::kHalf ? 1 : 2;
}

// an index tensor on the same device: int32 or int64
int index_i64(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what, ": int32 or int64");
  TORCH_CHECK(t.device() == like.device(), what, ": must be on ", like.device());
  return t.scalar_type() == at::kLong ? 1 : 0;
}

// ------------------------------------------------------------------ rotary --

std::vector<Tensor> rotary(Tensor q, OptTensor k, OptTensor pos, int64_t offset, Tensor inv, bool interleaved,
                           double scale, double sign) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && q.stride(3) == 1, "rotary: q (B, L, H, D) on the GPU, unit inner stride");
  c10::cuda::CUDAGuard guard(q.device());
  vagus::RotaryArgs a = {};
  a.B = q.size(0); a.L = q.size(1); a.H = static_cast<int>(q.size(2)); a.D = static_cast<int>(q.size(3));
  a.q = q.data_ptr();
  a.sq_b = q.stride(0); a.sq_l = q.stride(1); a.sq_h = q.stride(2);
  auto yq = torch::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  a.yq = yq.data_ptr();
  std::vector<Tensor> out = {yq};
  if (has(k)) {
    TORCH_CHECK(k->device() == q.device() && k->scalar_type() == q.scalar_type() && k->dim() == 4 &&
                    k->size(0) == a.B && k->size(1) == a.L && k->size(3) == a.D && k->stride(3) == 1,
                "rotary: k (B, L, Hk, D) like q");
    a.Hk = static_cast<int>(k->size(2));
    a.k = k->data_ptr();
    a.sk_b = k->stride(0); a.sk_l = k->stride(1); a.sk_h = k->stride(2);
    out.push_back(torch::empty(k->sizes(), k->options().memory_format(at::MemoryFormat::Contiguous)));
    a.yk = out[1].data_ptr();
  }
  if (has(pos)) {
    a.pos_i64 = index_i64(*pos, q, "rotary positions");
    TORCH_CHECK(pos->dim() == 2 && pos->size(0) == a.B && pos->size(1) == a.L, "rotary: positions (B, L)");
    a.pos = pos->data_ptr();
    a.pos_sb = pos->stride(0); a.pos_sl = pos->stride(1);
  }
  a.offset = offset;
  TORCH_CHECK(inv.scalar_type() == at::kDouble && inv.is_contiguous() && inv.dim() == 1 && inv.device() == q.device(),
              "rotary: inv_freq (R / 2) float64 on q's device");
  a.inv = inv.data_ptr<double>();
  a.R = static_cast<int>(2 * inv.size(0));
  a.interleaved = interleaved ? 1 : 0;
  a.scale = static_cast<float>(scale);
  a.sign = static_cast<float>(sign);
  check(vagus::rotary(a, type_of(q, "rotary"), at::cuda::getCurrentCUDAStream().stream()), "rotary");
  return out;
}

// ---------------------------------------------------------------- 4-bit KV --

struct Cache {
  Tensor kc, kp, vc, vp;
  int64_t B, Hk, cap, D, Dv;
};

Cache cache_of(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp) {
  TORCH_CHECK(kc.is_cuda() && kc.dim() == 4, "int4 cache: codes (B, Hk, capacity, D / 2) on the GPU");
  Cache c{kc, kp, vc, vp, kc.size(0), kc.size(1), kc.size(2), 2 * kc.size(3), 2 * vc.size(3)};
  for (const Tensor* t : {&kc, &kp, &vc, &vp})
    TORCH_CHECK(t->device() == kc.device() && t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "int4 cache: contiguous, 16-byte aligned tensors on one device");
  TORCH_CHECK(kc.scalar_type() == at::kByte && vc.scalar_type() == at::kByte && kp.scalar_type() == at::kBFloat16 &&
                  vp.scalar_type() == at::kBFloat16,
              "int4 cache: uint8 codes and bf16 parameters");
  TORCH_CHECK(vc.dim() == 4 && vc.size(0) == c.B && vc.size(1) == c.Hk && vc.size(2) == c.cap, "int4 cache: shapes");
  TORCH_CHECK(c.D % 32 == 0 && c.Dv % 32 == 0 && c.cap % 16 == 0 && c.cap < (int64_t(1) << 31) - 64,
              "int4 cache: head dims in groups of 32, capacity in blocks of 16");
  TORCH_CHECK(kp.sizes() == at::IntArrayRef({c.B, c.Hk, c.cap, c.D / 32, 2}) &&
                  vp.sizes() == at::IntArrayRef({c.B, c.Hk, c.cap, c.Dv / 32, 2}),
              "int4 cache: parameters (B, Hk, capacity, D / 32, 2)");
  return c;
}

// a start or length per sequence
void per_row(const OptTensor& t, const Cache& c, const void*& p, int& i64, const char* what) {
  if (!has(t)) return;
  i64 = index_i64(*t, c.kc, what);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == c.B && t->is_contiguous(), what, ": (B,) contiguous");
  p = t->data_ptr();
}

void kv4_append(Tensor kc, Tensor kp, Tensor vc, Tensor vp, Tensor k, Tensor v, OptTensor start, int64_t offset) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.device() == kc.device() && v.device() == kc.device() &&
                  k.scalar_type() == v.scalar_type() && k.stride(3) == 1 && v.stride(3) == 1,
              "kv4_append: k, v (B, Hk, L, D) of one type, unit inner stride");
  const int64_t L = k.size(2);
  TORCH_CHECK(k.sizes() == at::IntArrayRef({c.B, c.Hk, L, c.D}) && v.sizes() == at::IntArrayRef({c.B, c.Hk, L, c.Dv}),
              "kv4_append: k, v must match the cache");
  vagus::Kv4AppendArgs a = {};
  a.k = k.data_ptr(); a.v = v.data_ptr();
  a.sk_b = k.stride(0); a.sk_h = k.stride(1); a.sk_l = k.stride(2);
  a.sv_b = v.stride(0); a.sv_h = v.stride(1); a.sv_l = v.stride(2);
  a.k_codes = kc.data_ptr(); a.k_params = kp.data_ptr(); a.v_codes = vc.data_ptr(); a.v_params = vp.data_ptr();
  per_row(start, c, a.start, a.start_i64, "kv4_append start");
  TORCH_CHECK(a.start || (offset >= 0 && offset + L <= c.cap), "kv4_append: tokens [", offset, ", ", offset + L,
              ") leave the cache of ", c.cap);
  a.offset = offset;
  a.B = c.B; a.L = L; a.cap = c.cap; a.Hk = static_cast<int>(c.Hk); a.D = static_cast<int>(c.D);
  a.Dv = static_cast<int>(c.Dv);
  a.err = vagus_device_error_ptr();
  check(vagus::kv4_append(a, type_of(k, "kv4_append"), at::cuda::getCurrentCUDAStream().stream()), "kv4_append");
}

std::vector<Tensor> kv4_read(Tensor kc, Tensor kp, Tensor vc, Tensor vp, OptTensor start, int64_t offset,
                             int64_t count) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  vagus::Kv4ReadArgs a = {};
  per_row(start, c, a.start, a.start_i64, "kv4_read start");
  TORCH_CHECK(count >= 0 && (a.start || (offset >= 0 && offset + count <= c.cap)), "kv4_read: tokens [", offset, ", ",
              offset + count, ") leave the cache of ", c.cap);
  auto k = torch::empty({c.B, c.Hk, count, c.D}, kp.options()), v = torch::empty({c.B, c.Hk, count, c.Dv}, kp.options());
  a.k_codes = kc.data_ptr(); a.k_params = kp.data_ptr(); a.v_codes = vc.data_ptr(); a.v_params = vp.data_ptr();
  a.k = k.data_ptr(); a.v = v.data_ptr();
  a.offset = offset;
  a.B = c.B; a.L = count; a.cap = c.cap; a.Hk = static_cast<int>(c.Hk); a.D = static_cast<int>(c.D);
  a.Dv = static_cast<int>(c.Dv);
  a.err = vagus_device_error_ptr();
  check(vagus::kv4_read(a, at::cuda::getCurrentCUDAStream().stream()), "kv4_read");
  return {k, v};
}

// q (B, H, Lq, D) bf16 -> (B, H, Lq, Dv), token-major underneath like attn_fwd's
Tensor kv4_attn(Tensor q, Tensor kc, Tensor kp, Tensor vc, Tensor vp, OptTensor lengths, int64_t length, bool causal,
                double scale) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  TORCH_CHECK(q.dim() == 4 && q.device() == kc.device() && q.scalar_type() == at::kBFloat16 && q.size(0) == c.B &&
                  q.size(3) == c.D && c.Hk > 0 && q.size(1) % c.Hk == 0,
              "kv4_attn: q (B, H, Lq, D) bf16, H a multiple of the cache's heads");
  bool ok = q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && q.stride(d) % 8 == 0;
  if (!ok) q = q.clone(at::MemoryFormat::Contiguous);
  vagus::Kv4AttnArgs a = {};
  a.q = q.data_ptr();
  a.sq_b = q.stride(0); a.sq_h = q.stride(1); a.sq_l = q.stride(2);
  a.k_codes = static_cast<const unsigned char*>(kc.data_ptr());
  a.v_codes = static_cast<const unsigned char*>(vc.data_ptr());
  a.k_params = kp.data_ptr(); a.v_params = vp.data_ptr();
  per_row(lengths, c, a.lengths, a.len_i64, "kv4_attn lengths");
  TORCH_CHECK(a.lengths || (length >= 0 && length <= c.cap), "kv4_attn: ", length, " tokens in a cache of ", c.cap);
  a.length = length;
  a.B = c.B; a.cap = c.cap; a.H = static_cast<int>(q.size(1)); a.Hk = static_cast<int>(c.Hk);
  a.Lq = static_cast<int>(q.size(2)); a.D = static_cast<int>(c.D); a.Dv = static_cast<int>(c.Dv);
  a.causal = causal ? 1 : 0;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.err = vagus_device_error_ptr();
  auto o = torch::empty({c.B, q.size(2), q.size(1), c.Dv}, q.options().memory_format(at::MemoryFormat::Contiguous));
  a.o = o.data_ptr();
  a.splits = 1;
  Tensor part, ml;
  if (o.numel() > 0) {
    a.splits = vagus::kv4_attn_splits(a, a.lengths ? c.cap : length);
    if (a.splits > 1) {
      const auto f32 = q.options().dtype(at::kFloat);
      part = torch::empty({c.B, q.size(2), q.size(1), a.splits, c.Dv}, f32);
      ml = torch::empty({c.B, q.size(2), q.size(1), a.splits, 2}, f32);
      a.part_o = part.data_ptr<float>();
      a.part_ml = ml.data_ptr<float>();
    }
    check(vagus::kv4_attn(a, at::cuda::getCurrentCUDAStream().stream()), "kv4_attn");
  }
  return o.transpose(1, 2);
}

// ------------------------------------------------------------------ verify --

std::vector<Tensor> verify_draft(Tensor target, OptTensor draft, Tensor tokens, Tensor u_accept, Tensor u_sample,
                                 OptTensor lengths) {
  TORCH_CHECK(target.is_cuda() && target.dim() == 3 && target.stride(2) == 1 && target.size(1) >= 1,
              "verify_draft: target (B, K + 1, V) on the GPU, unit inner stride");
  c10::cuda::CUDAGuard guard(target.device());
  vagus::VerifyArgs a = {};
  a.B = target.size(0); a.V = target.size(2); a.K = static_cast<int>(target.size(1) - 1);
  a.target = target.data_ptr(); a.st_b = target.stride(0); a.st_k = target.stride(1);
  if (has(draft)) {
    TORCH_CHECK(draft->device() == target.device() && draft->scalar_type() == target.scalar_type() &&
                    draft->sizes() == at::IntArrayRef({a.B, static_cast<int64_t>(a.K), a.V}) && draft->stride(2) == 1,
                "verify_draft: draft (B, K, V) like the target");
    a.draft = draft->data_ptr(); a.sd_b = draft->stride(0); a.sd_k = draft->stride(1);
  }
  const std::vector<int64_t> bk = {a.B, a.K};
  TORCH_CHECK(tokens.device() == target.device() && tokens.scalar_type() == at::kLong && tokens.sizes() == bk,
              "verify_draft: tokens (B, K) int64");
  TORCH_CHECK(u_accept.device() == target.device() && u_accept.scalar_type() == at::kFloat && u_accept.sizes() == bk,
              "verify_draft: u_accept (B, K) fp32");
  TORCH_CHECK(u_sample.device() == target.device() && u_sample.scalar_type() == at::kFloat && u_sample.dim() == 1 &&
                  u_sample.size(0) == a.B,
              "verify_draft: u_sample (B,) fp32");
  tokens = tokens.contiguous();
  u_accept = u_accept.contiguous();
  u_sample = u_sample.contiguous();
  a.tokens = reinterpret_cast<const long long*>(tokens.data_ptr<int64_t>()); a.stok_b = a.K;
  a.u_accept = u_accept.data_ptr<float>(); a.su_b = a.K;
  a.u_sample = u_sample.data_ptr<float>();
  if (has(lengths)) {
    a.len_i64 = index_i64(*lengths, target, "verify_draft lengths");
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == a.B && lengths->is_contiguous(), "verify_draft: lengths (B,)");
    a.lengths = lengths->data_ptr();
  }
  auto out = torch::empty({a.B, a.K + 1}, tokens.options()), acc = torch::empty({a.B}, tokens.options());
  a.out = reinterpret_cast<long long*>(out.data_ptr<int64_t>());
  a.accepted = reinterpret_cast<long long*>(acc.data_ptr<int64_t>());
  check(vagus::verify_draft(a, type_of(target, "verify_draft"), at::cuda::getCurrentCUDAStream().stream()),
        "verify_draft");
  return {out, acc};
}

}  // namespace

void register_stream_ops(pybind11::module& m) {
  m.def("rotary", &rotary);
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attn", &kv4_attn);
  m.def("verify_draft", &verify_draft);
}
