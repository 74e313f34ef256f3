// Python binding of the serving-step operators: checks of the tensors, outputs and workspace, and one call of the C ABI
// (include/fgw_mha.h) per operator.
//
// Why it is compiled: these calls take 4 to 15 microseconds on the GPU when batches are small, and checking ten tensors,
// packing the parameters and calling through ctypes took 10 to 20 in Python; here it is about 2. The operators' contracts
// and messages are those of fgw_b200/operators/mha/{chunk_attention,rotary_append,page_ops}.py, which document them.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "fgw_mha.h"

namespace {

constexpr int64_t kInt32Max = 0x7fffffff;
constexpr int64_t kMaxGroup = 128;  // query heads that may share a key head

using Optional = std::optional<at::Tensor>;

void require(bool ok, const char* message) {
  if (!ok) throw pybind11::value_error(message);
}

// A non-zero status of the C ABI as the package's FgwError.
void check_status(int status, const char* call) {
  if (status == FGW_OK) return;
  const auto type = pybind11::module_::import("fgw_b200._native").attr("FgwError");
  const auto error = type(status, call);
  PyErr_SetObject(type.ptr(), error.ptr());
  throw pybind11::error_already_set();
}

void* stream_of(const at::Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

int dtype_code(at::ScalarType type) {
  return type == at::kBFloat16 ? FGW_DTYPE_BFLOAT16 : FGW_DTYPE_FLOAT16;
}

// The checks shared by the operators over a ragged batch and a paged cache.
struct Ragged {
  int64_t tokens, heads, dim, kv_heads, rows, batch, width;
};

Ragged check_ragged(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table,
                    const at::Tensor& lens, const at::Tensor& cu, int64_t page) {
  require(q.dim() == 3 && k_cache.dim() == 3 && v_cache.sizes() == k_cache.sizes(), "Expected q[T,H,D] and K/V[N,Hkv,D]");
  Ragged r;
  r.tokens = q.size(0);
  r.heads = q.size(1);
  r.dim = q.size(2);
  r.rows = k_cache.size(0);
  r.kv_heads = k_cache.size(1);
  require(k_cache.size(2) == r.dim && r.kv_heads > 0 && r.heads > 0 && r.heads % r.kv_heads == 0,
          "K/V heads must divide the query heads and share their dimension");
  const auto type = q.scalar_type();
  require((type == at::kHalf || type == at::kBFloat16) && k_cache.scalar_type() == type && v_cache.scalar_type() == type,
          "FP16 or BF16 required, the same for every tensor");
  require(r.dim >= 16 && r.dim <= 256 && r.dim % 16 == 0, "D must be in [16, 256] and divisible by 16");
  require(page > 0 && page % 16 == 0 && r.rows > 0 && r.rows % page == 0,
          "page_size must be a positive multiple of 16 and divide the pool's rows");
  require(table.dim() == 2 && lens.dim() == 1 && cu.dim() == 1, "metadata shape mismatch");
  r.batch = table.size(0);
  r.width = table.size(1);
  require(r.batch > 0 && r.width > 0 && lens.size(0) == r.batch && cu.size(0) == r.batch + 1, "metadata shape mismatch");
  require(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt && cu.scalar_type() == at::kInt,
          "page table, lengths and offsets must be int32");
  require(r.width <= kInt32Max / page && r.tokens <= kInt32Max && r.rows <= kInt32Max && r.batch <= kInt32Max &&
              r.heads <= kInt32Max,
          "requires logical positions, tokens and pool rows to fit int32");
  const auto device = q.device();
  require(device.is_cuda() && k_cache.device() == device && v_cache.device() == device && table.device() == device &&
              lens.device() == device && cu.device() == device,
          "every tensor must be on the same CUDA device");
  require(k_cache.is_contiguous() && v_cache.is_contiguous() && table.is_contiguous() && lens.is_contiguous() &&
              cu.is_contiguous(),
          "kernel inputs must be contiguous");
  return r;
}

// Elements from one token's row to the next of x [tokens, heads, dim]; each row itself is contiguous.
int64_t token_stride(const at::Tensor& x) {
  const int64_t tokens = x.size(0), heads = x.size(1), dim = x.size(2);
  require(x.stride(2) == 1 && (x.stride(1) == dim || heads <= 1), "a token's heads must be contiguous");
  if (tokens <= 1) return heads * dim;
  require(x.stride(0) >= heads * dim && x.stride(0) % 8 == 0,
          "the token stride must be a multiple of 8 and cover the heads");
  return x.stride(0);
}

// The data pointer, 16-byte aligned as the kernels' vector accesses and TMA need it.
void* aligned(const at::Tensor& x) {
  void* at = x.data_ptr();
  require(reinterpret_cast<uintptr_t>(at) % 16 == 0, "tensors must be 16-byte aligned");
  return at;
}

int32_t* ints(const at::Tensor& x) { return x.data_ptr<int32_t>(); }

// `out`, or a new contiguous tensor of q's shape.
at::Tensor output_like(const at::Tensor& q, const Optional& out) {
  if (!out.has_value()) return at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  require(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->device() == q.device(),
          "out must match q");
  return *out;
}

at::Tensor paged_chunk_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                 const at::Tensor& table, const at::Tensor& lens, const at::Tensor& cu, int64_t page,
                                 bool causal, std::optional<double> scale, const Optional& given) {
  const Ragged r = check_ragged(q, k_cache, v_cache, table, lens, cu, page);
  require(r.heads <= kMaxGroup * r.kv_heads, "at most 128 query heads per key head");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(r.dim));
  require(s > 0.0 && s <= 1e30 && static_cast<float>(s) > 0.f, "softmax_scale must be positive and finite");
  const int64_t q_stride = token_stride(q);
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor out = output_like(q, given);
  const int64_t out_stride = token_stride(out);
  if (r.tokens == 0) return out;
  fgw_chunk_params p = {};
  p.q = aligned(q);
  p.k_cache = aligned(k_cache);
  p.v_cache = aligned(v_cache);
  p.out = aligned(out);
  p.block_table = ints(table);
  p.cache_seqlens = ints(lens);
  p.cu_seqlens_q = ints(cu);
  p.tokens = r.tokens;
  p.pool_rows = r.rows;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.batch = static_cast<int32_t>(r.batch);
  p.heads = static_cast<int32_t>(r.heads);
  p.kv_heads = static_cast<int32_t>(r.kv_heads);
  p.head_dim = static_cast<int32_t>(r.dim);
  p.table_width = static_cast<int32_t>(r.width);
  p.page_size = static_cast<int32_t>(page);
  p.dtype = dtype_code(q.scalar_type());
  p.causal = causal ? 1 : 0;
  p.softmax_scale = static_cast<float>(s);
  size_t bytes = 0;
  check_status(fgw_chunk_workspace_size(&p, &bytes), "fgw_chunk_workspace_size");
  const at::Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  check_status(fgw_chunk_attention(&p, workspace.data_ptr(), bytes, stream_of(q)), "fgw_chunk_attention");
  return out;
}

at::Tensor rotary_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                         const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& cu,
                         const at::Tensor& cos_sin, int64_t page, bool interleaved, const Optional& given) {
  const Ragged r = check_ragged(q, k_cache, v_cache, table, lens, cu, page);
  require(k.dim() == 3 && k.size(0) == r.tokens && k.size(1) == r.kv_heads && k.size(2) == r.dim && v.sizes() == k.sizes(),
          "Expected k and v [T,Hkv,D]");
  require(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && cos_sin.scalar_type() == at::kFloat,
          "k and v take q's type, cos_sin float32");
  require(cos_sin.dim() == 2, "cos_sin must be [positions, rotary_dim]");
  const int64_t positions = cos_sin.size(0), rotary = cos_sin.size(1);
  require(positions > 0 && rotary >= 2 && rotary <= r.dim && rotary % 2 == 0,
          "cos_sin must have a row and rotary_dim be even and at most D");
  require(k.device() == q.device() && v.device() == q.device() && cos_sin.device() == q.device(),
          "every tensor must be on the same CUDA device");
  require(cos_sin.is_contiguous(), "kernel inputs must be contiguous");
  fgw_rotary_params p = {};
  p.q_stride = token_stride(q);
  p.k_stride = token_stride(k);
  p.v_stride = token_stride(v);
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor out = output_like(q, given);
  p.q_out_stride = token_stride(out);
  if (r.tokens == 0) return out;
  p.q = aligned(q);
  p.k = aligned(k);
  p.v = aligned(v);
  p.q_out = aligned(out);
  p.k_cache = aligned(k_cache);
  p.v_cache = aligned(v_cache);
  p.block_table = ints(table);
  p.cache_seqlens = ints(lens);
  p.cu_seqlens_q = ints(cu);
  p.cos_sin = cos_sin.data_ptr<float>();
  p.tokens = r.tokens;
  p.pool_rows = r.rows;
  p.batch = static_cast<int32_t>(r.batch);
  p.heads = static_cast<int32_t>(r.heads);
  p.kv_heads = static_cast<int32_t>(r.kv_heads);
  p.head_dim = static_cast<int32_t>(r.dim);
  p.rotary_dim = static_cast<int32_t>(rotary);
  p.positions = static_cast<int32_t>(std::min(positions, kInt32Max));
  p.table_width = static_cast<int32_t>(r.width);
  p.page_size = static_cast<int32_t>(page);
  p.dtype = dtype_code(q.scalar_type());
  p.interleaved = interleaved ? 1 : 0;
  check_status(fgw_rotary_append(&p, stream_of(q)), "fgw_rotary_append");
  return out;
}

// The pools' part of the parameters; `at` receives their pointers and outlives the call.
fgw_page_params check_pools(const std::vector<at::Tensor>& pools, int64_t page, std::vector<void*>& at) {
  require(!pools.empty(), "at least one pool required");
  const at::Tensor& first = pools[0];
  const int64_t rows = first.dim() >= 2 ? first.size(0) : 0;
  require(page > 0 && page <= kInt32Max && rows > 0 && rows % page == 0,
          "pools must be [num_pages * page_size, ...] with a positive page size");
  const int64_t row_bytes = first.numel() / rows * first.element_size();
  require(row_bytes > 0 && row_bytes % 16 == 0, "a pool row must be a multiple of 16 bytes");
  require(rows / page <= int64_t(1) << 30, "at most 2^30 pages");
  at.reserve(pools.size());
  for (const at::Tensor& pool : pools) {
    require(pool.sizes() == first.sizes() && pool.scalar_type() == first.scalar_type() && pool.device() == first.device(),
            "pools must have one shape, type and device");
    require(pool.is_cuda(), "every tensor must be on the same CUDA device");
    require(pool.is_contiguous(), "pools must be contiguous and 16-byte aligned");
    at.push_back(aligned(pool));
  }
  fgw_page_params p = {};
  p.pools = at.data();
  p.pool_count = static_cast<int32_t>(pools.size());
  p.row_bytes = row_bytes;
  p.page_size = static_cast<int32_t>(page);
  p.num_pages = static_cast<int32_t>(rows / page);
  return p;
}

void check_rows(const at::Tensor& x, const at::Tensor& pool) {
  require(x.scalar_type() == at::kInt, "page table, lengths and page lists must be int32");
  require(x.device() == pool.device(), "every tensor must be on the same CUDA device");
  require(x.is_contiguous(), "kernel inputs must be contiguous");
}

void check_table(const at::Tensor& table, const at::Tensor& lens, int64_t page, const at::Tensor& pool,
                 fgw_page_params& p) {
  require(table.dim() == 2 && lens.dim() == 1 && lens.size(0) == table.size(0) && table.numel() > 0,
          "metadata shape mismatch");
  require(table.size(1) <= kInt32Max / page && table.numel() <= FGW_PAGE_MAX_ENTRIES,
          "requires logical positions to fit int32 and at most 2^31 - 2^16 table entries");
  check_rows(table, pool);
  check_rows(lens, pool);
  p.block_table = ints(table);
  p.cache_seqlens = ints(lens);
  p.batch = static_cast<int32_t>(table.size(0));
  p.table_width = static_cast<int32_t>(table.size(1));
}

using PageCall = int (*)(const fgw_page_params*, void*, size_t, void*);

void run_pages(PageCall call, const char* name, const fgw_page_params& p, const at::Tensor& pool) {
  size_t bytes = 0;
  check_status(fgw_page_workspace_size(&p, &bytes), "fgw_page_workspace_size");
  const at::Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, pool.options().dtype(at::kByte));
  check_status(call(&p, workspace.data_ptr(), bytes, stream_of(pool)), name);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> fork_pages(const std::vector<at::Tensor>& pools, const at::Tensor& table,
                                                          const at::Tensor& lens, const at::Tensor& parents, int64_t page,
                                                          const Optional& reserve) {
  std::vector<void*> at;
  fgw_page_params p = check_pools(pools, page, at);
  check_table(table, lens, page, pools[0], p);
  require(parents.sizes() == lens.sizes() && (!reserve.has_value() || reserve->sizes() == lens.sizes()),
          "metadata shape mismatch");
  check_rows(parents, pools[0]);
  if (reserve.has_value()) check_rows(*reserve, pools[0]);
  const c10::cuda::CUDAGuard guard(pools[0].device());
  at::Tensor table_out = at::empty_like(table), lens_out = at::empty_like(lens), status = at::empty({2}, lens.options());
  p.parents = ints(parents);
  p.reserve_seqlens = reserve.has_value() ? ints(*reserve) : nullptr;
  p.table_out = ints(table_out);
  p.seqlens_out = ints(lens_out);
  p.status = ints(status);
  run_pages(fgw_page_fork, "fgw_page_fork", p, pools[0]);
  return {table_out, lens_out, status};
}

std::tuple<at::Tensor, at::Tensor> compact_pages(const std::vector<at::Tensor>& pools, const at::Tensor& table,
                                                 const at::Tensor& lens, int64_t page) {
  std::vector<void*> at;
  fgw_page_params p = check_pools(pools, page, at);
  check_table(table, lens, page, pools[0], p);
  const c10::cuda::CUDAGuard guard(pools[0].device());
  at::Tensor table_out = at::empty_like(table), status = at::empty({2}, lens.options());
  p.table_out = ints(table_out);
  p.status = ints(status);
  run_pages(fgw_page_compact, "fgw_page_compact", p, pools[0]);
  return {table_out, status};
}

void copy_pages(const std::vector<at::Tensor>& pools, const at::Tensor& src, const at::Tensor& dst, int64_t page) {
  std::vector<void*> at;
  fgw_page_params p = check_pools(pools, page, at);
  require(src.dim() == 1 && dst.sizes() == src.sizes() && src.numel() <= kInt32Max, "metadata shape mismatch");
  check_rows(src, pools[0]);
  check_rows(dst, pools[0]);
  if (src.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(pools[0].device());
  p.src_pages = ints(src);
  p.dst_pages = ints(dst);
  p.copy_count = static_cast<int32_t>(src.numel());
  run_pages(fgw_page_copy, "fgw_page_copy", p, pools[0]);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // the header this file was compiled with: its version, and the sizes of the structures it passes
  m.attr("built_for") = pybind11::make_tuple(FGW_MHA_ABI_VERSION, sizeof(fgw_chunk_params), sizeof(fgw_rotary_params),
                                             sizeof(fgw_page_params));
  m.def("paged_chunk_attention", &paged_chunk_attention);
  m.def("rotary_append", &rotary_append);
  m.def("fork_pages", &fork_pages);
  m.def("compact_pages", &compact_pages);
  m.def("copy_pages", &copy_pages);
}
