// Python bindings, fourth part: page pools that streams share. Launched on the current stream of the cache's device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <limits>

#include "api_shared.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

inline cudaStream_t cur_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
inline void check(int rc, const char* what) {
  if (rc == 0) return;
  if (rc > 0) TORCH_CHECK(false, what, ": CUDA error ", rc, " (", cudaGetErrorString((cudaError_t)rc), ")");
  TORCH_CHECK(rc != -2, what, ": more segments or rows than a call plans");
  TORCH_CHECK(false, what, ": unsupported arguments (code ", rc, ")");
}
bool aligned(const Tensor& t, int64_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }
bool bf16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16; }
bool f32(const Tensor& t) { return t.scalar_type() == torch::kFloat32; }
const int* ints(const Tensor& t, int64_t n, const Tensor& beside, const char* what, const char* name) {
  TORCH_CHECK(t.is_contiguous() && t.scalar_type() == torch::kInt32 && t.numel() == n && t.device() == beside.device(), what, ": ", name, " is not ", n,
              " int32 on the cache's device");
  return t.data_ptr<int>();
}

// k [pages, kv_block, nkv, hd] bf16, q [rows, nq, hd] bf16 with dense heads
FbSharedStep check_step(const Tensor& q, const Tensor& k, const Tensor& kvlen, const Tensor& table, int64_t kv_block, int64_t nq, int64_t nkv, int64_t hd,
                        const Tensor& seg_slot, const Tensor& seg_row0, const Tensor& seg_nrows, int64_t max_rows, const OptTensor& grp_seg0,
                        const OptTensor& grp_nsegs, const OptTensor& grp_len, const Tensor& status, const char* what) {
  TORCH_CHECK(nq > 0 && nkv > 0 && nq % nkv == 0 && nq / nkv <= 128, what, ": ", nq, " query heads over ", nkv, " (whole shares of up to 128)");
  TORCH_CHECK(hd == 64 || hd == 128 || hd == 256, what, ": heads of ", hd, " columns (64, 128 or 256)");
  TORCH_CHECK(kv_block > 0 && kv_block % 64 == 0, what, ": pages of ", kv_block, " tokens (multiples of 64)");
  TORCH_CHECK(k.is_cuda() && bf16(k) && k.is_contiguous() && k.dim() == 4 && k.size(1) == kv_block && k.size(2) == nkv && k.size(3) == hd && aligned(k, 16),
              what, ": cache is not [pages, ", kv_block, ", ", nkv, ", ", hd, "] bf16");
  TORCH_CHECK(k.size(0) > 0 && k.size(0) * kv_block < std::numeric_limits<int>::max(), what, ": pages of the pool");
  TORCH_CHECK(bf16(q) && q.dim() == 3 && q.size(1) == nq && q.size(2) == hd && (q.size(0) < 2 || q.stride(0) % 8 == 0) && q.stride(1) == hd &&
              q.stride(2) == 1 && aligned(q, 16) && q.device() == k.device(), what, ": q is not [rows, ", nq, ", ", hd, "] bf16 with dense heads");
  TORCH_CHECK(q.size(0) * nq < (1 << 30), what, ": rows");
  TORCH_CHECK(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 && table.size(1) * kv_block < std::numeric_limits<int>::max(), what, ": block_table");
  TORCH_CHECK(nkv * (table.size(1) * kv_block / 64 + 8) < std::numeric_limits<int>::max(), what, ": block_table of ", table.size(1) * kv_block, " tokens");
  TORCH_CHECK((max_rows >= 1 || seg_slot.numel() == 0 || q.size(0) == 0) && max_rows <= std::numeric_limits<int>::max() && status.scalar_type() == torch::kInt32 && status.device() == k.device(), what,
              ": max_rows, status");
  TORCH_CHECK(grp_seg0.has_value() == grp_nsegs.has_value() && grp_seg0.has_value() == grp_len.has_value(), what, ": groups");
  FbSharedStep st{};
  const int64_t S = seg_slot.numel();
  TORCH_CHECK(S <= 4096, what, ": ", S, " segments (4096 at most)");
  st.seg_slot = ints(seg_slot, S, k, what, "seg_slot");
  st.seg_row0 = ints(seg_row0, S, k, what, "seg_row0");
  st.seg_nrows = ints(seg_nrows, S, k, what, "seg_nrows");
  st.nseg = (int)S;
  st.max_rows = (int)max_rows;
  if (grp_seg0) {
    const int64_t G = grp_seg0->numel();
    TORCH_CHECK(G <= S, what, ": ", G, " groups of ", S, " segments");
    st.grp_seg0 = ints(*grp_seg0, G, k, what, "grp_seg0");
    st.grp_nsegs = ints(*grp_nsegs, G, k, what, "grp_nsegs");
    st.grp_len = ints(*grp_len, G, k, what, "grp_len");
    st.ngrp = (int)G;
  }
  st.kvlen = ints(kvlen, q.size(0), k, what, "row_kvlen");
  st.rows = (int)q.size(0);
  st.table = ints(table, table.numel(), k, what, "block_table");
  st.slots = (int)table.size(0);
  st.max_blocks = (int)table.size(1);
  st.kv_block = (int)kv_block;
  st.pages = (long)k.size(0);
  return st;
}

void attention_shared(Tensor out, OptTensor lse, Tensor ws, Tensor q, Tensor k, Tensor v, OptTensor proj, Tensor kvlen, Tensor table, int64_t kv_block,
                      int64_t nq, int64_t nkv, int64_t hd, Tensor seg_slot, Tensor seg_row0, Tensor seg_nrows, int64_t max_rows, OptTensor grp_seg0,
                      OptTensor grp_nsegs, OptTensor grp_len, int64_t ctas, Tensor status) {
  const char* what = "attention_shared";
  const FbSharedStep st = check_step(q, k, kvlen, table, kv_block, nq, nkv, hd, seg_slot, seg_row0, seg_nrows, max_rows, grp_seg0, grp_nsegs, grp_len,
                                     status, what);
  const int64_t T = q.size(0);
  TORCH_CHECK(bf16(v) && v.is_contiguous() && v.sizes() == k.sizes() && v.device() == k.device() && aligned(v, 16), what, ": v_cache is not like k_cache");
  TORCH_CHECK(bf16(out) && out.is_contiguous() && out.numel() == T * nq * hd && out.device() == k.device() && aligned(out, 16), what, ": out");
  TORCH_CHECK(!lse || (f32(*lse) && lse->is_contiguous() && lse->numel() == T * nq && lse->device() == k.device()), what, ": lse");
  TORCH_CHECK(!proj || (bf16(*proj) && proj->dim() == 2 && proj->size(0) == T && proj->size(1) >= 2 * nq * hd && proj->stride(1) == 1 &&
                        proj->device() == k.device()), what, ": proj is not [rows, at least ", 2 * nq * hd, "] bf16");
  TORCH_CHECK(f32(ws) && ws.is_contiguous() && ws.device() == k.device() && aligned(ws, 16), what, ": workspace");
  const c10::cuda::CUDAGuard guard(k.device());
  check(fb_attention_shared(out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr<float>(), (long)ws.numel(), q.data_ptr(), (long)q.stride(0),
                            k.data_ptr(), v.data_ptr(), proj ? proj->data_ptr() : nullptr, proj ? (long)proj->stride(0) : 0, st, (int)nq, (int)nkv, (int)hd,
                            (int)ctas, status.data_ptr<int>(), cur_stream()), what);
}

int64_t attention_mass(Tensor out, Tensor mass, double carry, OptTensor lse, Tensor ws, Tensor q, Tensor k, Tensor kvlen, Tensor table, int64_t kv_block,
                    int64_t nq, int64_t nkv, int64_t hd, Tensor seg_slot, Tensor seg_row0, Tensor seg_nrows, int64_t max_rows, OptTensor grp_seg0,
                    OptTensor grp_nsegs, OptTensor grp_len, int64_t ctas, Tensor status) {
  const char* what = "attention_mass";
  const FbSharedStep st = check_step(q, k, kvlen, table, kv_block, nq, nkv, hd, seg_slot, seg_row0, seg_nrows, max_rows, grp_seg0, grp_nsegs, grp_len,
                                     status, what);
  TORCH_CHECK(nq / nkv <= 64, what, ": ", nq, " query heads over ", nkv, " (shares of up to 64)");
  for (const Tensor& t : {out, mass})
    TORCH_CHECK(f32(t) && t.is_contiguous() && t.dim() == 3 && t.size(0) == k.size(0) && t.size(1) == nkv && t.size(2) == kv_block &&
                t.device() == k.device(), what, ": sums are not [pages, ", nkv, ", ", kv_block, "] fp32");
  TORCH_CHECK(!lse || (f32(*lse) && lse->is_contiguous() && lse->numel() == q.size(0) * nq && lse->device() == k.device()), what, ": lse is not [rows, ", nq,
              "] fp32");
  TORCH_CHECK(f32(ws) && ws.is_contiguous() && ws.device() == k.device() && aligned(ws, 16), what, ": workspace");
  const c10::cuda::CUDAGuard guard(k.device());
  check(fb_attention_mass(out.data_ptr<float>(), mass.data_ptr<float>(), (float)carry, lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr<float>(),
                          (long)ws.numel(), q.data_ptr(), (long)q.stride(0), k.data_ptr(), st, (int)nq, (int)nkv, (int)hd, (int)ctas,
                          status.data_ptr<int>(), cur_stream()), what);
  return fb_attention_mass_launches(st.rows, st.nseg, st.max_rows, st.ngrp, (int)nq, (int)nkv, (int)hd, !lse);
}

// k, v [pages, kv_block, nkv, ..] of 16-bit values or of codes; scale [pages, kv_block, nkv, ns]
void kv_evict(Tensor kept, Tensor k, Tensor v, OptTensor scale, Tensor mass, Tensor seg_slot, Tensor seg_len, Tensor table, Tensor dst, int64_t kv_block,
              int64_t keep, int64_t first, int64_t recent, int64_t ctas, Tensor status) {
  const char* what = "kv_evict";
  TORCH_CHECK(k.is_cuda() && k.is_contiguous() && k.dim() == 4 && kv_block > 0 && k.size(1) == kv_block && k.size(0) > 0 &&
              k.size(0) * kv_block < std::numeric_limits<int>::max() && aligned(k, 16), what, ": cache is not [pages, ", kv_block, ", kv heads, ..]");
  TORCH_CHECK(v.is_contiguous() && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device() && aligned(v, 16), what,
              ": v_cache is not like k_cache");
  const int64_t nkv = k.size(2), row = k.size(3) * k.element_size(), S = seg_slot.numel();
  TORCH_CHECK(nkv > 0 && row > 0 && row % 16 == 0 && row <= (1 << 20), what, ": rows of ", row, " bytes a head (multiples of 16)");
  TORCH_CHECK(!scale || (f32(*scale) && scale->is_contiguous() && scale->dim() == 4 && scale->size(0) == k.size(0) && scale->size(1) == kv_block &&
                         scale->size(2) == nkv && scale->size(3) > 0 && scale->size(3) <= 32 && scale->device() == k.device()), what,
              ": kv_scale is not [pages, ", kv_block, ", ", nkv, ", up to 32] fp32");
  TORCH_CHECK(f32(mass) && mass.is_contiguous() && mass.dim() == 3 && mass.size(0) == k.size(0) && mass.size(1) == nkv && mass.size(2) == kv_block &&
              mass.device() == k.device(), what, ": sums are not [pages, ", nkv, ", ", kv_block, "] fp32");
  TORCH_CHECK(keep > 0 && first >= 0 && recent >= 0 && first <= keep && recent <= keep - first, what, ": first ", first, " and recent ", recent, " of ", keep);
  TORCH_CHECK(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 && table.size(1) * kv_block < std::numeric_limits<int>::max(), what, ": block_table");
  TORCH_CHECK(dst.dim() == 2 && dst.size(0) == S && dst.size(1) * kv_block >= keep && dst.size(1) * kv_block < std::numeric_limits<int>::max(), what,
              ": dst_table is not [segments, pages for ", keep, " tokens]");
  TORCH_CHECK(S * nkv * keep < std::numeric_limits<int>::max(), what, ": segments");
  TORCH_CHECK(kept.is_contiguous() && kept.scalar_type() == torch::kInt32 && kept.numel() == S * nkv * keep && kept.device() == k.device(), what, ": kept");
  TORCH_CHECK(status.scalar_type() == torch::kInt32 && status.device() == k.device(), what, ": status");
  const c10::cuda::CUDAGuard guard(k.device());
  check(fb_kv_evict(kept.data_ptr<int>(), k.data_ptr(), v.data_ptr(), scale ? scale->data_ptr<float>() : nullptr, mass.data_ptr<float>(),
                    ints(seg_slot, S, k, what, "seg_slot"), ints(seg_len, S, k, what, "seg_len"), (int)S, ints(table, table.numel(), k, what, "block_table"),
                    (int)table.size(0), (int)table.size(1), ints(dst, dst.numel(), k, what, "dst_table"), (int)dst.size(1), (long)k.size(0), (int)kv_block,
                    (int)nkv, (int)row, scale ? (int)scale->size(3) : 0, (int)keep, (int)first, (int)recent, (int)ctas, status.data_ptr<int>(),
                    cur_stream()), what);
}

}  // namespace

void register_shared(pybind11::module_& m) {
  m.def("attention_shared", &attention_shared);
  m.def("attention_shared_floats", &fb_attention_shared_floats);
  m.def("attention_mass", &attention_mass);
  m.def("attention_mass_floats", &fb_attention_mass_floats);
  m.def("kv_evict", &kv_evict);
}
