// Python bindings of the 4-bit KV cache: writer, reader, paged attention, page copies.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cfloat>
#include <cstdlib>
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "kv_fp4.h"
#include "paged_attention_fp4.h"

namespace {

constexpr double kLog2e = 1.4426950408889634;

int64_t page_bytes(int64_t d) { return 64 * (d / 2 + d / 16); }

void check_dim(int64_t d, const char* who) {
  TORCH_CHECK(d == 64 || d == 128 || d == 256, who, ": head_dim 64, 128 or 256, got ", d);
}

void check_cache(const torch::Tensor& k, const torch::Tensor& v, int64_t d, const char* who) {
  for (const torch::Tensor* c : {&k, &v})
    TORCH_CHECK(c->is_cuda() && c->scalar_type() == at::kByte && c->dim() == 3 && c->is_contiguous() &&
                    c->size(2) == page_bytes(d),
                who, ": caches uint8 [num_blocks, kv_heads, ", page_bytes(d), "] contiguous on a CUDA device");
  for (const torch::Tensor* c : {&k, &v})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(c->data_ptr()) % 16 == 0, who, ": caches must be 16-byte aligned");
  TORCH_CHECK(k.sizes() == v.sizes() && k.device() == v.device(), who, ": key and value caches of one shape on one device");
  TORCH_CHECK(k.size(0) > 0 && k.size(0) <= 0x7fffffff, who, ": 1 .. 2^31 - 1 blocks");
}

// A cache's scale and its reciprocal are kept as normal fp32 numbers.
void check_scales(double k_scale, double v_scale, const char* who) {
  for (const double s : {k_scale, v_scale})
    TORCH_CHECK(s >= FLT_MIN && s <= 1.0 / FLT_MIN, who, ": cache scales must be positive, from 2^-126 to 2^126, got ", s);
}

void check_index(const torch::Tensor& t, at::ScalarType type, int64_t dim, const torch::Tensor& like, const char* who,
                 const char* name) {
  TORCH_CHECK(t.scalar_type() == type && t.dim() == dim && t.device() == like.device(), who, ": ", name, " must be ",
              c10::toString(type), " with ", dim, " dimension(s) on ", like.device());
  TORCH_CHECK(t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1, who, ": ", name, " must have unit stride");
}

void check_rows(const torch::Tensor& t, int64_t width, const torch::Tensor& like, const char* who, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.device() == like.device(), who,
              ": ", name, " must be bf16 [tokens, width] on ", like.device());
  TORCH_CHECK(t.size(1) >= width && (t.size(1) <= 1 || t.stride(1) == 1), who, ": ", name, " needs ", width,
              " columns of unit stride");
  TORCH_CHECK(t.size(0) == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                                 (t.size(0) == 1 || t.stride(0) % 8 == 0)),
              who, ": ", name, " rows must be 16-byte aligned");
}

// Partial results and tickets of the split units, one set per stream: calls on a stream follow one another, calls on
// two streams may overlap.  A capture has sets of its own, so that a replay never shares one with eager calls, and one for
// each of its streams, for the branches of a graph may overlap too.  They live in the graph's pool; a set's tickets are
// zeroed by a node of the graph, on the stream that the set belongs to.  The sets of a device's last capture are kept until
// another one asks (one that is still open gets new ones then: the old memory is only reused behind its own stream's work).
struct Scratch {
  torch::Tensor part, tickets;
};
struct CaptureScratch {
  unsigned long long id = 0;
  std::map<cudaStream_t, Scratch> sets;
};

Scratch scratch(const torch::Tensor& like, cudaStream_t stream, int64_t floats, int64_t ctas) {
  static std::mutex mu;
  static auto* eager = new std::map<std::pair<int, cudaStream_t>, Scratch>();  // never destroyed: outlives CUDA
  static auto* captured = new std::map<int, CaptureScratch>();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  TORCH_CHECK(cudaStreamGetCaptureInfo(stream, &status, &id) == cudaSuccess, "paged_attention_fp4: stream capture state");
  std::lock_guard<std::mutex> lock(mu);
  const int dev = like.get_device();
  Scratch* s;
  if (status == cudaStreamCaptureStatusActive) {
    CaptureScratch& capture = (*captured)[dev];
    if (capture.id != id) {
      capture.sets.clear();
      capture.id = id;
    }
    s = &capture.sets[stream];
  } else {
    s = &(*eager)[{dev, stream}];
  }
  if (!s->part.defined() || s->part.numel() < floats)
    s->part = torch::empty({floats}, like.options().dtype(at::kFloat));
  if (!s->tickets.defined() || s->tickets.numel() < ctas)
    s->tickets = torch::zeros({ctas}, like.options().dtype(at::kInt));
  return *s;
}

}  // namespace

torch::Tensor rope_kv_write_fp4(const torch::Tensor& qkv, const torch::Tensor& positions, const torch::Tensor& cos_sin,
                                const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& slots,
                                int64_t hq, int64_t hk, int64_t d, int64_t rot, double k_scale, double v_scale,
                                const c10::optional<torch::Tensor>& out) {
  const char* who = "rope_kv_write_fp4";
  check_dim(d, who);
  check_cache(k_cache, v_cache, d, who);
  TORCH_CHECK(hq > 0 && hk > 0 && k_cache.size(1) == hk, who, ": the caches hold ", k_cache.size(1), " kv heads, not ", hk);
  check_rows(qkv, (hq + 2 * hk) * d, k_cache, who, "qkv");
  const torch::Tensor q_out = out.has_value() ? *out : torch::empty({qkv.size(0), hq * d}, qkv.options());
  check_rows(q_out, hq * d, k_cache, who, "q_out");
  TORCH_CHECK(q_out.size(0) == qkv.size(0), who, ": one q_out row per token");
  TORCH_CHECK(!q_out.is_alias_of(qkv), who, ": q_out must not share qkv's memory (a rotation reads both halves)");
  check_index(positions, at::kLong, 1, k_cache, who, "positions");
  check_index(slots, at::kLong, 1, k_cache, who, "slot_mapping");
  TORCH_CHECK(positions.numel() == qkv.size(0) && slots.numel() == qkv.size(0), who, ": one position and slot per token");
  TORCH_CHECK(rot >= 0 && rot <= d && rot % 2 == 0, who, ": rot must be even and at most head_dim");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2 && cos_sin.size(1) == rot &&
                  cos_sin.is_contiguous() && cos_sin.device() == k_cache.device() && cos_sin.size(0) > 0,
              who, ": cos_sin must be f32 [positions, rot] contiguous");
  check_scales(k_scale, v_scale, who);
  if (qkv.size(0) == 0) return q_out;
  const c10::cuda::CUDAGuard guard(k_cache.device());
  KvFp4WriteParams p{};
  p.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.qkv_stride = qkv.size(0) == 1 ? 0 : qkv.stride(0);
  p.q_out = reinterpret_cast<__nv_bfloat16*>(q_out.data_ptr());
  p.q_stride = qkv.size(0) == 1 ? 0 : q_out.stride(0);
  p.positions = positions.data_ptr<int64_t>();
  p.cos_sin = cos_sin.data_ptr<float>();
  p.max_pos = cos_sin.size(0);
  p.slots = slots.data_ptr<int64_t>();
  p.k_cache = k_cache.data_ptr<uint8_t>();
  p.v_cache = v_cache.data_ptr<uint8_t>();
  p.num_tokens = qkv.size(0);
  p.num_slots = k_cache.size(0) * 64;
  p.hq = static_cast<int>(hq);
  p.hk = static_cast<int>(hk);
  p.rot = static_cast<int>(rot);
  p.k_inv = static_cast<float>(1.0 / k_scale);
  p.v_inv = static_cast<float>(1.0 / v_scale);
  const int r = sh_kv_fp4_write(&p, static_cast<int>(d), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(r == 0, "sh_kv_fp4_write failed with code ", r);
  return q_out;
}

std::tuple<torch::Tensor, torch::Tensor> kv_fp4_read(const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                                     const torch::Tensor& slots, int64_t d, double k_scale,
                                                     double v_scale) {
  const char* who = "kv_fp4_read";
  check_dim(d, who);
  check_cache(k_cache, v_cache, d, who);
  check_index(slots, at::kLong, 1, k_cache, who, "slots");
  check_scales(k_scale, v_scale, who);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const auto options = k_cache.options().dtype(at::kBFloat16);
  const torch::Tensor k_out = torch::empty({slots.numel(), k_cache.size(1), d}, options);
  const torch::Tensor v_out = torch::empty({slots.numel(), k_cache.size(1), d}, options);
  if (slots.numel() == 0) return {k_out, v_out};
  KvFp4ReadParams p{};
  p.k_cache = k_cache.data_ptr<uint8_t>();
  p.v_cache = v_cache.data_ptr<uint8_t>();
  p.k_out = reinterpret_cast<__nv_bfloat16*>(k_out.data_ptr());
  p.v_out = reinterpret_cast<__nv_bfloat16*>(v_out.data_ptr());
  p.slots = slots.data_ptr<int64_t>();
  p.n = slots.numel();
  p.num_slots = k_cache.size(0) * 64;
  p.hk = static_cast<int>(k_cache.size(1));
  p.k_scale = static_cast<float>(k_scale);
  p.v_scale = static_cast<float>(v_scale);
  const int r = sh_kv_fp4_read(&p, static_cast<int>(d), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(r == 0, "sh_kv_fp4_read failed with code ", r);
  return {k_out, v_out};
}

void paged_attention_fp4(const torch::Tensor& out, const torch::Tensor& q, const torch::Tensor& k_cache,
                         const torch::Tensor& v_cache, const torch::Tensor& block_tables, const torch::Tensor& seq_lens,
                         const torch::Tensor& q_start, int64_t hq, int64_t d, double scale, int64_t max_q_len,
                         double k_scale, double v_scale, const c10::optional<torch::Tensor>& err) {
  const char* who = "paged_attention_fp4";
  const char* env = std::getenv("SH_BATCH_INVARIANT");
  const bool invariant = env != nullptr && env[0] == '1' && env[1] == 0;
  check_dim(d, who);
  check_cache(k_cache, v_cache, d, who);
  const int64_t hk = k_cache.size(1), B = seq_lens.numel();
  TORCH_CHECK(hk > 0 && hq > 0 && hq % hk == 0, who, ": ", hq, " query heads over ", hk, " kv heads");
  check_rows(q, hq * d, k_cache, who, "q");
  check_rows(out, hq * d, k_cache, who, "out");
  TORCH_CHECK(out.size(0) == q.size(0), who, ": one out row per q row");
  check_index(block_tables, at::kInt, 2, k_cache, who, "block_tables");
  check_index(seq_lens, at::kLong, 1, k_cache, who, "seq_lens");
  check_index(q_start, at::kLong, 1, k_cache, who, "q_start");
  TORCH_CHECK(q_start.numel() == B + 1 && block_tables.size(0) == B, who, ": q_start of ", B + 1, " and block_tables of ",
              B, " rows for ", B, " lengths");
  TORCH_CHECK(max_q_len >= 1, who, ": max_q_len must be at least 1");
  check_scales(k_scale, v_scale, who);
  TORCH_CHECK(!err.has_value() || (err->scalar_type() == at::kInt && err->numel() >= 1 && err->device() == k_cache.device()),
              who, ": err must be int32 on ", k_cache.device());
  if (q.size(0) == 0 || B == 0) return;
  TORCH_CHECK(block_tables.size(1) > 0, who, ": block_tables without columns");
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  AttnFp4Params p{};
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.out_stride = out.size(0) == 1 ? 0 : out.stride(0);
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_stride = q.size(0) == 1 ? 0 : q.stride(0);
  p.k_cache = k_cache.data_ptr<uint8_t>();
  p.v_cache = v_cache.data_ptr<uint8_t>();
  p.block_tables = block_tables.data_ptr<int32_t>();
  p.bt_stride = block_tables.stride(0);
  p.seq_lens = seq_lens.data_ptr<int64_t>();
  p.q_start = q_start.data_ptr<int64_t>();
  p.err = err.has_value() ? err->data_ptr<int>() : nullptr;
  p.num_tokens = q.size(0);
  p.B = static_cast<int>(B);
  p.hq = static_cast<int>(hq);
  p.hk = static_cast<int>(hk);
  p.num_blocks = static_cast<int>(k_cache.size(0));
  p.bt_cols = static_cast<int>(std::min<int64_t>(block_tables.size(1), (1 << 25) - 1));  // positions fit an int
  p.whole_units = invariant ? 1 : 0;
  p.scale_log2 = static_cast<float>(scale * k_scale * kLog2e);
  p.v_scale = static_cast<float>(v_scale);
  const int dim = static_cast<int>(d);
  const int64_t rows = std::min<int64_t>(max_q_len, 4096) * (hq / hk);  // of one kv head
  int r;
  // The tensor-core kernel takes units of 256 rows (128 at head_dim 256) whatever they hold, and starts up in 10 to
  // 20 us; the other one's time grows with its row tiles, and a lone request's keys are spread over fewer warps.  Short
  // kernel against this one, in us:
  //   rows: 32 requests of 6000 keys on average, head_dim 128, 100 against 172 at 32 rows, 173 against 173 at 36 and 48;
  //     24 of 3000 at head_dim 256, 48 against 49 at 48, 58 against 49 at 64, 67 against 49 at 72;
  //   keys, one request with 32 heads of 128: 12 against 21 for a prompt of 200, 29 against 21 for one of 300, 27 against
  //     21 for 16 tokens at 1000, 80 against 54 for 17 at 30000;
  //   work (query rows times keys at most), one request, 16 heads of 256: 17 against 20 for a prompt of 160 (0.5M), 32
  //     against 39 for 17 tokens at 8000 (2.2M), 32 against 25 for a prompt of 400 (2.9M), 121 against 42 for one of 1000
  //     (16M); 8 heads of 64: 10 against 18 for 400 (1.4M), 29 against 39 for 64 tokens at 12000 (6.2M), 31 against 22 for
  //     1000 (8.2M).
  // Keys are the table's columns, for no length is known on the host.  A table far wider than its lengths, as decode steps
  // pass, makes short windows of many rows look large: 7 tokens at head_dim 256 over 200 keys take 28 where a tight table
  // gives 14 (4 requests) and 23 (24 requests); over 1000 keys 34 against 24, and 42 against 42.
  const int64_t keys = int64_t{64} * p.bt_cols;
  const double work = static_cast<double>(q.size(0)) * static_cast<double>(hq) * static_cast<double>(keys);
  const bool large = d == 128 ? keys > 256 || work > 4e6 : work > (d == 256 ? 2.5e6 : 7.5e6);
  if (rows > (d == 256 ? 48 : 32) && large && !invariant) {
    const int64_t floats = sh_paged_attention_fp4_tc_workspace(dim);
    TORCH_CHECK(floats > 0, who, ": no CUDA device");
    const Scratch s = scratch(k_cache, stream, floats, 0);
    p.part_o = s.part.data_ptr<float>();
    r = sh_paged_attention_fp4_tc(&p, dim, stream);
  } else {
    // Rows that a CTA holds: as many as the longest query has, up to what its registers carry.  Tiles of different
    // sizes deal the keys to their warps differently, so batch-invariant calls always take the largest.
    const int most = d == 256 ? 16 : 32;
    const int tile = invariant ? most : static_cast<int>(std::min<int64_t>((rows + 7) / 8 * 8, most));
    const int ctas = sh_paged_attention_fp4_ctas(dim, tile);
    TORCH_CHECK(ctas > 0, who, ": no CUDA device");
    const Scratch s = scratch(k_cache, stream, sh_paged_attention_fp4_workspace(dim, tile), ctas);
    p.part_o = s.part.data_ptr<float>();
    p.tickets = reinterpret_cast<unsigned*>(s.tickets.data_ptr<int>());
    r = sh_paged_attention_fp4(&p, dim, tile, stream);
  }
  TORCH_CHECK(r == 0, "sh_paged_attention_fp4 failed with code ", r);
}

// The list is walked in place: an engine passes two tensors a layer, and a copy of each would cost as much as the call.
void copy_kv_pages(const py::list& caches, const torch::Tensor& src, const torch::Tensor& dst) {
  const char* who = "copy_kv_pages";
  const Py_ssize_t count = PyList_GET_SIZE(caches.ptr());
  auto cache = [&](Py_ssize_t i) -> const at::Tensor& {
    PyObject* o = PyList_GET_ITEM(caches.ptr(), i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), who, ": caches must be tensors");
    return THPVariable_Unpack(o);
  };
  TORCH_CHECK(count > 0 && cache(0).is_cuda(), who, ": at least one CUDA cache tensor");
  const c10::Device device = cache(0).device();
  check_index(src, at::kLong, 1, cache(0), who, "src");
  check_index(dst, at::kLong, 1, cache(0), who, "dst");
  TORCH_CHECK(src.numel() == dst.numel(), who, ": ", src.numel(), " sources for ", dst.numel(), " destinations");
  std::vector<KvCopyParams> calls((count + SH_KV_COPY_MAX_TENSORS - 1) / SH_KV_COPY_MAX_TENSORS);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor& c = cache(i);
    TORCH_CHECK(c.device() == device && c.dim() >= 2 && c.is_contiguous(), who,
                ": cache tensors [num_blocks, ...] contiguous on one device");
    const int64_t n = c.numel();
    if (n == 0) continue;
    const int64_t bytes = n / c.size(0) * static_cast<int64_t>(c.element_size());
    uint8_t* base = static_cast<uint8_t*>(c.data_ptr());
    TORCH_CHECK(bytes % 16 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0, who,
                ": pages must be multiples of 16 bytes and 16-byte aligned");
    KvCopyParams& p = calls[i / SH_KV_COPY_MAX_TENSORS];
    p.base[p.tensors] = base;
    p.page_bytes[p.tensors] = bytes;
    p.pages[p.tensors] = c.size(0);
    ++p.tensors;
  }
  if (src.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  for (KvCopyParams& p : calls) {
    p.src = src.data_ptr<int64_t>();
    p.dst = dst.data_ptr<int64_t>();
    p.n = src.numel();
    const int r = sh_kv_copy_pages(&p, stream);
    TORCH_CHECK(r == 0, "sh_kv_copy_pages failed with code ", r);
  }
}
