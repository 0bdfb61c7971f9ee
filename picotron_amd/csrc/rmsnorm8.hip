// C ABI of RMSNorm with an 8-bit checkpoint (kernels in rmsnorm8_impl.hpp), and the kernel that joins the partial rows of dw.
#include "rmsnorm8_impl.hpp"

namespace pt {
namespace rmsnorm8 {

extern template int launch<float>(bool, bool, bool, const Norm8&, void*, hipStream_t);
extern template int launch<_Float16>(bool, bool, bool, const Norm8&, void*, hipStream_t);
extern template int launch<__bf16>(bool, bool, bool, const Norm8&, void*, hipStream_t);

// Adds the partial rows: 32 columns a workgroup, 32 threads a column.
__global__ __launch_bounds__(1024) void norm8_dw_kernel(const float* __restrict__ parts, int64_t count, int cols, void* __restrict__ dw,
                                                        int dtype) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x % 32, p = threadIdx.x / 32, col = blockIdx.x * 32 + c;
  float sum = 0.f;
  if (col < cols)
    for (int64_t k = p; k < count; k += 32) sum += parts[k * cols + col];
  sums[p][c] = sum;
  __syncthreads();
  if (p == 0 && col < cols) {
    for (int k = 1; k < 32; ++k) sum += sums[k][c];
    store_any(dw, col, dtype, sum);
  }
}

int join_dw(const float* parts, int64_t count, int cols, void* dw, int dtype, hipStream_t st) {
  hipLaunchKernelGGL(norm8_dw_kernel, dim3(static_cast<unsigned>((cols + 31) / 32)), dim3(1024), 0, st, parts, count, cols, dw, dtype);
  return check_launch("pt_rmsnorm8_bwd");
}

}  // namespace rmsnorm8

namespace {

int by_type(bool backward, const rmsnorm8::Norm8& a, void* dw, int dtype, hipStream_t st) {
  const bool aligned = aligned16(a.x) && aligned16(a.extra) && aligned16(a.h) && aligned16(a.y) && a.cols * dtype_size(dtype) % 16 == 0;
  const bool nt = a.rows * a.cols * dtype_size(dtype) > (int64_t{1} << 25);
  switch (dtype) {
    case PT_FLOAT32:
      return rmsnorm8::launch<float>(backward, aligned, nt, a, dw, st);
    case PT_FLOAT16:
      return rmsnorm8::launch<_Float16>(backward, aligned, nt, a, dw, st);
    default:
      return rmsnorm8::launch<__bf16>(backward, aligned, nt, a, dw, st);
  }
}

int check_norm8(const std::string& name, int64_t rows, int64_t cols, int x_dtype, int w_dtype, std::initializer_list<const void*> elements,
                const void* weight, const void* codes, const float* steps) {
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype)) return fail(PT_EUNSUPPORTED, name + ": dtype must be fp32, fp16 or bf16");
  if (rows < 0 || cols < 1) return fail(PT_EINVAL, name + ": bad sizes");
  if (rows > (int64_t{1} << 31) - 1 || cols > (int64_t{1} << 24)) return fail(PT_EUNSUPPORTED, name + ": under 2^31 rows of at most 2^24");
  if (rows == 0) return PT_OK;
  if (weight == nullptr || codes == nullptr || steps == nullptr) return fail(PT_EINVAL, name + ": null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 8 != 0 || reinterpret_cast<uintptr_t>(steps) % 4 != 0)
    return fail(PT_EINVAL, name + ": codes must be 8-byte aligned, steps 4-byte aligned");
  for (const void* p : elements)
    if (reinterpret_cast<uintptr_t>(p) % dtype_size(x_dtype) != 0) return fail(PT_EINVAL, name + ": misaligned pointer");
  if (reinterpret_cast<uintptr_t>(weight) % dtype_size(w_dtype) != 0) return fail(PT_EINVAL, name + ": misaligned pointer");
  return PT_OK;
}

}  // namespace
}  // namespace pt

extern "C" {

int pt_rmsnorm8_fwd(const void* x, const void* residual, const void* weight, void* h, void* y, float* rstd, void* codes, float* steps,
                    int64_t rows, int64_t cols, float eps, int x_dtype, int w_dtype, void* stream) {
  const std::string name("pt_rmsnorm8_fwd");
  if (int rc = pt::check_norm8(name, rows, cols, x_dtype, w_dtype, {x, residual, h, y}, weight, codes, steps)) return rc;
  if (rows == 0) return pt::ok();
  if (x == nullptr || y == nullptr || rstd == nullptr || (residual == nullptr) != (h == nullptr))
    return pt::fail(PT_EINVAL, name + ": null pointer, or a residual without its sum");
  pt::rmsnorm8::Norm8 a{};
  a.x = x;
  a.extra = residual;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.h = h;
  a.y = y;
  a.rstd = rstd;
  a.codes = static_cast<pt::block8::u32x2*>(codes);
  a.steps = steps;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.blocks = static_cast<int>((cols + pt::block8::kBlock - 1) / pt::block8::kBlock);
  a.eps = eps;
  return pt::by_type(false, a, nullptr, x_dtype, pt::as_stream(stream));
}

size_t pt_rmsnorm8_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  return static_cast<size_t>(pt::rmsnorm8::part_rows(rows, cols)) * static_cast<size_t>(cols) * 4;
}

int pt_rmsnorm8_bwd(const void* dy, const void* dh, const void* weight, const float* rstd, const void* codes, const float* steps, void* dx,
                    void* dweight, void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols, int x_dtype, int w_dtype, void* stream) {
  const std::string name("pt_rmsnorm8_bwd");
  if (int rc = pt::check_norm8(name, rows, cols, x_dtype, w_dtype, {dy, dh, dx}, weight, codes, steps)) return rc;
  if (dx == nullptr && dweight == nullptr) return pt::ok();
  hipStream_t st = pt::as_stream(stream);
  if (rows == 0) return dweight == nullptr ? pt::ok() : pt::fill(dweight, cols, pt::dtype_size(w_dtype), 0, st);
  if (dy == nullptr || rstd == nullptr) return pt::fail(PT_EINVAL, name + ": null pointer");
  if (dweight != nullptr && (workspace == nullptr || workspace_bytes < pt_rmsnorm8_bwd_workspace_bytes(rows, cols)))
    return pt::fail(PT_EINVAL, name + ": workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0 || reinterpret_cast<uintptr_t>(dweight) % pt::dtype_size(w_dtype) != 0)
    return pt::fail(PT_EINVAL, name + ": misaligned pointer");
  pt::rmsnorm8::Norm8 a{};
  a.x = dy;
  a.extra = dx != nullptr ? dh : nullptr;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.y = dx;
  a.rstd = const_cast<float*>(rstd);
  a.codes = static_cast<pt::block8::u32x2*>(const_cast<void*>(codes));
  a.steps = const_cast<float*>(steps);
  a.parts = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.blocks = static_cast<int>((cols + pt::block8::kBlock - 1) / pt::block8::kBlock);
  return pt::by_type(true, a, dweight, x_dtype, st);
}

}  // extern "C"
