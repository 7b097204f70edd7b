// Bindings of the long-context streaming operators: rotary positions
// (rotary.cu), the 4-bit key / value cache and attention over it (kv4.cu) and
// the verification of drafted tokens (verify.cu).  Every op runs on its
// tensors' device, on that device's current stream.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <string>
#include <tuple>
#include <vector>

#include "kernels.h"

int* vagus_device_error_ptr();   // bindings.cpp

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// Messages are built as strings: streaming a number into one (what the check
// macros do with their other arguments) needs the C++ library's locale facets,
// which a process with two C++ libraries may not have initialised.
std::string str(int64_t v) { return std::to_string(v); }
std::string str(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + ")";
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "vagus_b200 kernel '" + std::string(what) + "' rejected the problem or failed to launch (code " +
                           str(rc) + ")");
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

// an uninitialised dense tensor, without a trip through the dispatcher (a microsecond a call)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

int type_of(const Tensor& t, const char* what) {
  const auto s = t.scalar_type();
  TORCH_CHECK_VALUE(s == at::kFloat || s == at::kHalf || s == at::kBFloat16, std::string(what) + ": fp32, fp16 or bf16");
  return s == at::kFloat ? 0 : s == at::kHalf ? 1 : 2;
}

// an index tensor on the same device: int32 or int64
int index_i64(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, std::string(what) + ": int32 or int64");
  TORCH_CHECK_VALUE(t.device() == like.device(), std::string(what) + ": must be on the device of the other tensors");
  return t.scalar_type() == at::kLong ? 1 : 0;
}

// ------------------------------------------------------------------ rotary --

Tensor unit(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// pos: (L,) or (B, L), or none: token l sits at offset + l
std::tuple<Tensor, OptTensor> rotary(Tensor q, OptTensor k, OptTensor pos, int64_t offset, Tensor inv, bool interleaved,
                           double scale, double sign) {
  TORCH_CHECK_VALUE(q.is_cuda() && q.dim() == 4, "rotary: q (B, L, H, D)");
  c10::cuda::CUDAGuard guard(q.device());
  q = unit(q);
  vagus::RotaryArgs a = {};
  a.B = q.size(0); a.L = q.size(1); a.H = static_cast<int>(q.size(2)); a.D = static_cast<int>(q.size(3));
  a.q = q.data_ptr();
  a.sq_b = q.stride(0); a.sq_l = q.stride(1); a.sq_h = q.stride(2);
  Tensor yq = fresh({a.B, a.L, a.H, a.D}, q.scalar_type(), q);
  OptTensor yk;
  a.yq = yq.data_ptr();
  if (has(k)) {
    TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == a.B && k->size(1) == a.L && k->size(3) == a.D,
                      "rotary: q (B, L, H, D) and k (B, L, Hk, D)");
    TORCH_CHECK_VALUE(k->device() == q.device() && k->scalar_type() == q.scalar_type(),
                      "rotary: q and k must share dtype and device");
    k = unit(*k);
    a.Hk = static_cast<int>(k->size(2));
    a.k = k->data_ptr();
    a.sk_b = k->stride(0); a.sk_l = k->stride(1); a.sk_h = k->stride(2);
    yk = fresh({a.B, a.L, a.Hk, a.D}, q.scalar_type(), q);
    a.yk = yk->data_ptr();
  }
  if (has(pos)) {
    a.pos_i64 = index_i64(*pos, q, "rotary: positions");
    const bool per_token = pos->dim() == 1;
    TORCH_CHECK_VALUE((per_token || (pos->dim() == 2 && pos->size(0) == a.B)) && pos->size(-1) == a.L,
                      "rotary: positions of shape (L,) or (B, L)");
    a.pos = pos->data_ptr();
    a.pos_sb = per_token ? 0 : pos->stride(0);
    a.pos_sl = pos->stride(-1);
  }
  a.offset = offset;
  TORCH_CHECK_VALUE(inv.dim() == 1 && inv.is_floating_point() && inv.size(0) >= 1 && inv.size(0) <= a.D / 2 &&
                        inv.device() == q.device(),
                    "rotary: inv_freq (R/2,) on q's device with 2 <= R <= " + str(a.D));
  TORCH_CHECK_VALUE(inv.size(0) <= 4096, "rotary: R up to 8192 on the GPU");
  if (inv.scalar_type() != at::kDouble) inv = inv.to(at::kDouble);
  inv = inv.contiguous();
  a.inv = inv.data_ptr<double>();
  a.R = static_cast<int>(2 * inv.size(0));
  a.interleaved = interleaved ? 1 : 0;
  a.scale = static_cast<float>(scale);
  a.sign = static_cast<float>(sign);
  check(vagus::rotary(a, type_of(q, "rotary"), at::cuda::getCurrentCUDAStream().stream()), "rotary");
  return {yq, yk};
}

// ---------------------------------------------------------------- 4-bit KV --

struct Cache {
  Tensor kc, kp, vc, vp;
  int64_t B, Hk, cap, D, Dv;
};

Cache cache_of(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp) {
  TORCH_CHECK_VALUE(kc.is_cuda() && kc.dim() == 4 && vc.dim() == 4 && kp.dim() == 5 && vp.dim() == 5,
                    "Int4KV: codes (B, Hk, capacity, D / 2) and parameters (B, Hk, capacity, D / 32, 2)");
  Cache c{kc, kp, vc, vp, kc.size(0), kc.size(1), kc.size(2), 2 * kc.size(3), 2 * vc.size(3)};
  for (const Tensor* t : {&kc, &kp, &vc, &vp})
    TORCH_CHECK_VALUE(t->device() == kc.device() && t->is_contiguous() && t->size(0) == c.B && t->size(1) == c.Hk &&
                          t->size(2) == c.cap && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                      "Int4KV: contiguous, 16-byte aligned tensors of one batch, heads and capacity on one device");
  TORCH_CHECK_VALUE(kc.scalar_type() == at::kByte && vc.scalar_type() == at::kByte &&
                        kp.scalar_type() == at::kBFloat16 && vp.scalar_type() == at::kBFloat16,
                    "Int4KV: uint8 codes and bf16 parameters");
  TORCH_CHECK_VALUE(c.D > 0 && c.Dv > 0 && c.D % 32 == 0 && c.Dv % 32 == 0 && kp.size(3) == c.D / 32 &&
                        vp.size(3) == c.Dv / 32 && kp.size(4) == 2 && vp.size(4) == 2,
                    "Int4KV: head dims in groups of 32 with two parameters each");
  TORCH_CHECK_VALUE(c.D <= 4096 && c.Dv <= 4096, "Int4KV: head dims up to 4096 on the GPU");
  TORCH_CHECK_VALUE(c.cap % 16 == 0 && c.cap < (int64_t(1) << 30),
                    "Int4KV: the capacity must be a multiple of 16, below 2^30");
  return c;
}

// a start or length per sequence
void per_row(OptTensor& t, const Cache& c, const void*& p, int& i64, const char* what) {
  if (!has(t)) return;
  i64 = index_i64(*t, c.kc, what);
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == c.B, std::string(what) + ": (" + str(c.B) + ",)");
  t = t->contiguous();
  p = t->data_ptr();
}

void kv4_append(Tensor kc, Tensor kp, Tensor vc, Tensor vp, Tensor k, Tensor v, OptTensor start, int64_t offset) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.device() == kc.device() && v.device() == kc.device() &&
                        k.scalar_type() == v.scalar_type(),
                    "int4_append: k and v must share a dtype and be on the cache's device");
  const int64_t L = k.size(2);
  TORCH_CHECK_VALUE(k.size(0) == c.B && k.size(1) == c.Hk && k.size(3) == c.D && v.size(0) == c.B &&
                        v.size(1) == c.Hk && v.size(2) == L && v.size(3) == c.Dv,
                    "int4_append: k " + str(k.sizes()) + ", v " + str(v.sizes()) + " do not fit the cache");
  const int type = type_of(k, "int4_append");
  k = unit(k);
  v = unit(v);
  vagus::Kv4AppendArgs a = {};
  a.k = k.data_ptr(); a.v = v.data_ptr();
  a.sk_b = k.stride(0); a.sk_h = k.stride(1); a.sk_l = k.stride(2);
  a.sv_b = v.stride(0); a.sv_h = v.stride(1); a.sv_l = v.stride(2);
  a.k_codes = kc.data_ptr(); a.k_params = kp.data_ptr(); a.v_codes = vc.data_ptr(); a.v_params = vp.data_ptr();
  per_row(start, c, a.start, a.start_i64, "int4_append: start");
  TORCH_CHECK_VALUE(a.start || (offset >= 0 && L <= c.cap && offset <= c.cap - L), "int4_append: " + str(L) +
                    " tokens from " + str(offset) + " on leave the cache of " + str(c.cap));
  a.offset = offset;
  a.B = c.B; a.L = L; a.cap = c.cap; a.Hk = static_cast<int>(c.Hk); a.D = static_cast<int>(c.D);
  a.Dv = static_cast<int>(c.Dv);
  a.err = vagus_device_error_ptr();
  check(vagus::kv4_append(a, type, at::cuda::getCurrentCUDAStream().stream()), "kv4_append");
}

std::tuple<Tensor, Tensor> kv4_read(Tensor kc, Tensor kp, Tensor vc, Tensor vp, OptTensor start, int64_t offset,
                             int64_t count) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  vagus::Kv4ReadArgs a = {};
  per_row(start, c, a.start, a.start_i64, "int4_read: start");
  TORCH_CHECK_VALUE(count >= 0 && (a.start || (offset >= 0 && count <= c.cap && offset <= c.cap - count)), "int4_read: " +
                    str(count) + " tokens from " + str(offset) + " on leave the cache of " + str(c.cap));
  auto k = fresh({c.B, c.Hk, count, c.D}, at::kBFloat16, kc), v = fresh({c.B, c.Hk, count, c.Dv}, at::kBFloat16, kc);
  a.k_codes = kc.data_ptr(); a.k_params = kp.data_ptr(); a.v_codes = vc.data_ptr(); a.v_params = vp.data_ptr();
  a.k = k.data_ptr(); a.v = v.data_ptr();
  a.offset = offset;
  a.B = c.B; a.L = count; a.cap = c.cap; a.Hk = static_cast<int>(c.Hk); a.D = static_cast<int>(c.D);
  a.Dv = static_cast<int>(c.Dv);
  a.err = vagus_device_error_ptr();
  check(vagus::kv4_read(a, at::cuda::getCurrentCUDAStream().stream()), "kv4_read");
  return {k, v};
}

// q (B, H, Lq, D) -> (B, H, Lq, Dv), token-major underneath like attn_fwd's;
// none where no kernel serves the type or the head dims
c10::optional<Tensor> kv4_attn(Tensor q, Tensor kc, Tensor kp, Tensor vc, Tensor vp, OptTensor lengths, int64_t length,
                               bool causal) {
  const Cache c = cache_of(kc, kp, vc, vp);
  c10::cuda::CUDAGuard guard(kc.device());
  TORCH_CHECK_VALUE(q.dim() == 4 && q.device() == kc.device() && q.size(0) == c.B && q.size(3) == c.D && c.Hk > 0 &&
                        q.size(1) % c.Hk == 0,
                    "int4_attention: q " + str(q.sizes()) + " does not fit the cache");
  vagus::Kv4AttnArgs a = {};
  per_row(lengths, c, a.lengths, a.len_i64, "int4_attention: lengths");
  TORCH_CHECK_VALUE(a.lengths || (length >= 0 && length <= c.cap), "int4_attention: " + str(length) +
                    " tokens in a cache of " + str(c.cap));
  if (q.scalar_type() != at::kBFloat16 || (c.D != 64 && c.D != 128) || (c.Dv != 64 && c.Dv != 128))
    return c10::nullopt;
  bool ok = q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && q.stride(d) > 0 && q.stride(d) % 8 == 0;       // tensor maps take no stride of zero
  if (!ok) q = q.clone(at::MemoryFormat::Contiguous);
  a.q = q.data_ptr();
  a.sq_b = q.stride(0); a.sq_h = q.stride(1); a.sq_l = q.stride(2);
  a.k_codes = static_cast<const unsigned char*>(kc.data_ptr());
  a.v_codes = static_cast<const unsigned char*>(vc.data_ptr());
  a.k_params = kp.data_ptr(); a.v_params = vp.data_ptr();
  a.length = length;
  a.B = c.B; a.cap = c.cap; a.H = static_cast<int>(q.size(1)); a.Hk = static_cast<int>(c.Hk);
  a.Lq = static_cast<int>(q.size(2)); a.D = static_cast<int>(c.D); a.Dv = static_cast<int>(c.Dv);
  a.causal = causal ? 1 : 0;
  a.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(c.D)));
  a.err = vagus_device_error_ptr();
  auto o = fresh({c.B, q.size(2), q.size(1), c.Dv}, at::kBFloat16, q);
  a.o = o.data_ptr();
  Tensor part;
  if (vagus::kv4_attn_unpack_first(a)) {
    auto kv = kv4_read(kc, kp, vc, vp, c10::nullopt, 0, length);
    const Tensor &k = std::get<0>(kv), &v = std::get<1>(kv);
    auto lse = fresh({c.B, q.size(1), q.size(2)}, at::kFloat, q);
    vagus::AttnArgs f;
    f.q = a.q; f.k = k.data_ptr(); f.v = v.data_ptr(); f.o = a.o; f.lse = lse.data_ptr<float>();
    f.B = a.B; f.H = a.H; f.Hk = a.Hk; f.Lq = a.Lq; f.Lk = static_cast<int>(length); f.D = a.D; f.Dv = a.Dv;
    f.sq_b = a.sq_b; f.sq_h = a.sq_h; f.sq_l = a.sq_l;
    f.sk_b = k.stride(0); f.sk_h = k.stride(1); f.sk_l = k.stride(2);
    f.sv_b = v.stride(0); f.sv_h = v.stride(1); f.sv_l = v.stride(2);
    f.so_b = o.stride(0); f.so_h = o.stride(2); f.so_l = o.stride(1);
    f.causal = a.causal;
    f.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(c.D)));
    f.err = a.err;
    check(vagus::attn_fwd(f, at::cuda::getCurrentCUDAStream().stream()), "attn_fwd");
  } else if (o.numel() > 0) {
    check(vagus::kv4_attn_plan(a, a.lengths ? c.cap : length), "kv4_attn");
    if (a.part_rows > 0) {
      part = fresh({a.part_rows * (c.Dv + 2)}, at::kFloat, q);
      a.part_o = part.data_ptr<float>();
      a.part_ml = a.part_o + a.part_rows * c.Dv;
    }
    check(vagus::kv4_attn(a, at::cuda::getCurrentCUDAStream().stream()), "kv4_attn");
  }
  return o.transpose(1, 2);
}

// ------------------------------------------------------------------ verify --

std::tuple<Tensor, Tensor> verify_draft(Tensor target, OptTensor draft, Tensor tokens, Tensor u_accept, Tensor u_sample,
                                 OptTensor lengths) {
  TORCH_CHECK_VALUE(target.is_cuda() && target.dim() == 3 && target.size(1) >= 1 && target.size(2) >= 1,
                    "verify_draft: target (B, K + 1, V), fp32, fp16 or bf16");
  const int type = type_of(target, "verify_draft: target");
  c10::cuda::CUDAGuard guard(target.device());
  target = unit(target);
  vagus::VerifyArgs a = {};
  a.B = target.size(0); a.V = target.size(2); a.K = static_cast<int>(target.size(1) - 1);
  a.target = target.data_ptr(); a.st_b = target.stride(0); a.st_k = target.stride(1);
  if (has(draft)) {
    TORCH_CHECK_VALUE(draft->device() == target.device() && draft->scalar_type() == target.scalar_type() &&
                    draft->dim() == 3 && draft->size(0) == a.B && draft->size(1) == a.K && draft->size(2) == a.V,
                "verify_draft: draft (B, K, V) of the target's dtype");
    draft = unit(*draft);
    a.draft = draft->data_ptr(); a.sd_b = draft->stride(0); a.sd_k = draft->stride(1);
  }
  const std::vector<int64_t> bk = {a.B, a.K};
  TORCH_CHECK_VALUE(tokens.device() == target.device() && tokens.scalar_type() == at::kLong && tokens.sizes() == bk,
              "verify_draft: tokens (B, K) int64");
  TORCH_CHECK_VALUE(u_accept.device() == target.device() && u_accept.scalar_type() == at::kFloat && u_accept.sizes() == bk,
              "verify_draft: u_accept (B, K) fp32");
  TORCH_CHECK_VALUE(u_sample.device() == target.device() && u_sample.scalar_type() == at::kFloat && u_sample.dim() == 1 &&
                  u_sample.size(0) == a.B,
              "verify_draft: u_sample (B,) fp32");
  tokens = tokens.contiguous();
  u_accept = u_accept.contiguous();
  u_sample = u_sample.contiguous();
  a.tokens = reinterpret_cast<const long long*>(tokens.data_ptr<int64_t>()); a.stok_b = a.K;
  a.u_accept = u_accept.data_ptr<float>(); a.su_b = a.K;
  a.u_sample = u_sample.data_ptr<float>();
  if (has(lengths)) {
    a.len_i64 = index_i64(*lengths, target, "verify_draft: lengths");
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == a.B, "verify_draft: lengths (B,)");
    lengths = lengths->contiguous();
    a.lengths = lengths->data_ptr();
  }
  auto out = fresh({a.B, a.K + 1}, at::kLong, tokens), acc = fresh({a.B}, at::kLong, tokens);
  a.out = reinterpret_cast<long long*>(out.data_ptr<int64_t>());
  a.accepted = reinterpret_cast<long long*>(acc.data_ptr<int64_t>());
  check(vagus::verify_draft(a, type, at::cuda::getCurrentCUDAStream().stream()),
        "verify_draft");
  return {out, acc};
}

}  // namespace

void register_stream_ops(pybind11::module& m) {
  m.def("rotary", &rotary);
  m.def("kv4_check", [](Tensor kc, Tensor kp, Tensor vc, Tensor vp) {
    cache_of(kc, kp, vc, vp);
    c10::cuda::CUDAGuard guard(kc.device());
    vagus_device_error_ptr();             // made here, so that the first use may be captured into a graph
  });
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attn", &kv4_attn);
  m.def("verify_draft", &verify_draft);
}
