// Dropout without a stored mask (K12): y = keep * x / (1 - p), the same
// kernel forwards on x and backwards on dy.
//
// Bound by memory, one read and one write of each element: forward and
// backward over 47.8M bf16 take 78 us (4.9 TB/s), over 268M fp16 440 us (4.88);
// a large copy reaches 5.12. A stored mask would add a byte to the 4 of each
// element and direction. The generator needs 20 64-bit products, a quarter of
// the rate, for a block of four elements: by count 60 % of that time, behind
// the loads. Below a few million elements the host's launches are the bound
// (256 x 4096: 27 us for two kernels of 3).

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "philox.h"

namespace dvgg {

static inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

// 16-bit types: 8 elements (two blocks of the generator) a lane and step.
template <class T>
__global__ __launch_bounds__(256) void dropout16_kernel(
    const u16* __restrict__ x, u16* __restrict__ y, i64 n, DropArgs d,
    i64* __restrict__ used) {
  const u32 off = d.off();
  if (used && blockIdx.x == 0 && threadIdx.x == 0) *used = i64(off);
  for (i64 c = (i64)blockIdx.x * 256 + threadIdx.x; c < n / 8;
       c += (i64)gridDim.x * 256) {
    s16x8 v = *reinterpret_cast<const s16x8*>(x + c * 8);
    u32 k = keep4(d, off, 2 * c) | keep4(d, off, 2 * c + 1) << 4;
    s16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = (k >> j & 1) ? short(from_f(to_f(u16(v[j]), T()) * d.scale, T()))
                          : short(0);
    *reinterpret_cast<s16x8*>(y + c * 8) = o;
  }
  i64 i = n / 8 * 8 + threadIdx.x;
  if (blockIdx.x == 0 && i < n) {
    u32 k = keep4(d, off, i >> 2);
    y[i] = (k >> (i & 3) & 1) ? from_f(to_f(x[i], T()) * d.scale, T())
                              : u16(0);
  }
}

__global__ __launch_bounds__(256) void dropout32_kernel(
    const float* __restrict__ x, float* __restrict__ y, i64 n, DropArgs d,
    i64* __restrict__ used) {
  const u32 off = d.off();
  if (used && blockIdx.x == 0 && threadIdx.x == 0) *used = i64(off);
  for (i64 c = (i64)blockIdx.x * 256 + threadIdx.x; c < n / 4;
       c += (i64)gridDim.x * 256) {
    f32x4 v = *reinterpret_cast<const f32x4*>(x + c * 4);
    u32 k = keep4(d, off, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (k >> j & 1) ? v[j] * d.scale : 0.f;
    *reinterpret_cast<f32x4*>(y + c * 4) = v;
  }
  i64 i = n / 4 * 4 + threadIdx.x;
  if (blockIdx.x == 0 && i < n) {
    u32 k = keep4(d, off, i >> 2);
    y[i] = (k >> (i & 3) & 1) ? x[i] * d.scale : 0.f;
  }
}

// x: contiguous bf16, fp16 or fp32. offset_t: None, or one int64 on x's
// device that takes the place of `offset`; the kernel copies the value that
// it drew with into `used` for the backward pass.
std::vector<at::Tensor> dropout(const at::Tensor& x_, double p, int64_t seed,
                                int64_t offset,
                                const c10::optional<at::Tensor>& offset_t) {
  TORCH_CHECK(x_.is_cuda() && x_.is_contiguous(),
              "dropout: x must be a contiguous GPU tensor");
  auto type = x_.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf ||
              type == at::kFloat, "dropout: x must be bf16, fp16 or fp32, got ",
              type);
  TORCH_CHECK(p > 0.0 && p < 1.0, "dropout: p must lie in (0, 1), got ", p);
  const i64* offset_ptr = nullptr;
  if (offset_t) {
    TORCH_CHECK(offset_t->device() == x_.device() &&
                offset_t->scalar_type() == at::kLong &&
                offset_t->numel() == 1,
                "dropout: offset must be one int64 on x's device");
    offset_ptr = reinterpret_cast<const i64*>(offset_t->data_ptr<int64_t>());
  }
  c10::DeviceGuard guard(x_.device());
  // vector loads want 16-byte rows; a view that starts elsewhere is moved
  at::Tensor x = reinterpret_cast<uintptr_t>(x_.data_ptr()) % 16
                     ? x_.clone() : x_;
  auto y = at::empty_like(x);
  at::Tensor used;
  i64* used_ptr = nullptr;
  if (offset_t) {
    used = at::empty({1}, x.options().dtype(at::kLong));
    used_ptr = reinterpret_cast<i64*>(used.data_ptr<int64_t>());
  }
  i64 n = x.numel();
  DropArgs d = drop_args(p, seed, offset, offset_ptr);
  if (n > 0) {
    bool wide = type == at::kFloat;
    i64 chunks = wide ? n / 4 : n / 8;
    dim3 grid(u32(std::min<i64>(std::max<i64>((chunks + 255) / 256, 1),
                                4096)));
    auto stream = cur_stream();
    if (wide) {
      hipLaunchKernelGGL(dropout32_kernel, grid, dim3(256), 0, stream,
                         x.data_ptr<float>(), y.data_ptr<float>(), n, d,
                         used_ptr);
    } else {
      auto xp = reinterpret_cast<const u16*>(x.data_ptr());
      auto yp = reinterpret_cast<u16*>(y.data_ptr());
      if (type == at::kHalf)
        hipLaunchKernelGGL(dropout16_kernel<_Float16>, grid, dim3(256), 0,
                           stream, xp, yp, n, d, used_ptr);
      else
        hipLaunchKernelGGL(dropout16_kernel<__bf16>, grid, dim3(256), 0,
                           stream, xp, yp, n, d, used_ptr);
    }
    HIP_CHECK(hipGetLastError());
  } else if (offset_t) {
    used.zero_();
  }
  if (offset_t) return {y, used};
  return {y};
}

}  // namespace dvgg
