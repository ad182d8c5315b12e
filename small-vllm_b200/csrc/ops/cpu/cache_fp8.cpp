// CPU kernels of the 8-bit KV cache's operators on torch's thread pool: the rotary step that
// quantises as it writes, the read-back, and decode attention. fp32 inside (the scores' sums in 64
// bits), rounded once.
#include <ATen/Parallel.h>
#include <c10/util/BFloat16.h>
#include <c10/util/Exception.h>
#include <c10/util/Float8_e4m3fn.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <vector>

#include "ops/cache_fp8_kernels.h"
#include "ops/rope_kernels.h"

namespace svllm::ops::cpu_impl {
namespace {

using Code = c10::Float8_e4m3fn;

constexpr int kScaleMin = -60, kScaleMax = 60, kScaleBias = 127;
constexpr float kLargest = 448.0f;  // of e4m3
constexpr uint8_t kNanCode = 0x7f;

// One row of n values as codes and the e8m0 byte of its scale.
void quantise(const float* x, int64_t n, Code* codes, uint8_t* scale) {
  float amax = 0.0f;
  for (int64_t i = 0; i < n; ++i) {
    if (std::isfinite(x[i])) amax = std::max(amax, std::fabs(x[i]));
  }
  int e = kScaleMin;
  if (amax > 0.0f) {
    const float m = std::frexp(amax, &e);  // amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = std::clamp(e - (m <= 0.875f ? 9 : 8), kScaleMin, kScaleMax);
  }
  const float f = std::ldexp(1.0f, -e);
  for (int64_t i = 0; i < n; ++i) {
    codes[i] = std::isfinite(x[i]) ? Code(std::clamp(x[i] * f, -kLargest, kLargest))
                                   : Code(kNanCode, Code::from_bits());
  }
  *scale = static_cast<uint8_t>(e + kScaleBias);
}

float scale_value(uint8_t byte) { return std::ldexp(1.0f, static_cast<int>(byte) - kScaleBias); }

// The norm (where there is a weight) and rotation of one head in fp32.
void rotate(const at::BFloat16* x, const at::BFloat16* w, int64_t dim, float eps, const float* c,
            const float* s, float* y) {
  for (int64_t i = 0; i < dim; ++i) y[i] = static_cast<float>(x[i]);
  if (w != nullptr) {
    float sum = 0.0f;
    for (int64_t i = 0; i < dim; ++i) sum += y[i] * y[i];
    const float inv = 1.0f / std::sqrt(sum / static_cast<float>(dim) + eps);
    for (int64_t i = 0; i < dim; ++i) y[i] = y[i] * inv * static_cast<float>(w[i]);
  }
  for (int64_t i = 0; i < dim / 2; ++i) {
    const float a = y[i], b = y[i + dim / 2];
    y[i] = a * c[i] - b * s[i];
    y[i + dim / 2] = b * c[i] + a * s[i];
  }
}

}  // namespace

int64_t rope_cache_fp8(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& q_weight, const at::Tensor& k_weight,
                       const at::Tensor& positions, const at::Tensor& slot_mapping,
                       const at::Tensor& k_cache, const at::Tensor& v_cache,
                       const at::Tensor& k_scale, const at::Tensor& v_scale, double eps,
                       const float* inv_freq) {
  const int64_t tokens = q.size(0), heads = q.size(1), kv_heads = k.size(1), dim = q.size(2);
  const int64_t half = dim / 2, num_slots = k_scale.numel() / kv_heads;
  auto* qp = q.mutable_data_ptr<at::BFloat16>();
  const auto* kp = k.const_data_ptr<at::BFloat16>();
  const auto* vp = v.const_data_ptr<at::BFloat16>();
  const bool norm = q_weight.defined();
  const at::BFloat16* qw = norm ? q_weight.const_data_ptr<at::BFloat16>() : nullptr;
  const at::BFloat16* kw = norm ? k_weight.const_data_ptr<at::BFloat16>() : nullptr;
  const bool pos64 = positions.scalar_type() == at::kLong;
  const void* pos = positions.const_data_ptr();
  const auto* slots = slot_mapping.const_data_ptr<int64_t>();
  auto* kc = static_cast<Code*>(k_cache.mutable_data_ptr());
  auto* vc = static_cast<Code*>(v_cache.mutable_data_ptr());
  auto* ks = static_cast<uint8_t*>(k_scale.mutable_data_ptr());
  auto* vs = static_cast<uint8_t*>(v_scale.mutable_data_ptr());
  const float eps_f = static_cast<float>(eps);

  at::parallel_for(0, tokens, 16, [&](int64_t begin, int64_t end) {
    std::vector<float> c(half), s(half), y(dim);
    for (int64_t t = begin; t < end; ++t) {
      const double p = pos64 ? static_cast<double>(static_cast<const int64_t*>(pos)[t])
                             : static_cast<double>(static_cast<const int32_t*>(pos)[t]);
      for (int64_t i = 0; i < half; ++i) {
        const double angle = p * static_cast<double>(inv_freq[i]);
        c[i] = static_cast<float>(std::cos(angle));
        s[i] = static_cast<float>(std::sin(angle));
      }
      for (int64_t h = 0; h < heads; ++h) {
        at::BFloat16* x = qp + t * q.stride(0) + h * dim;
        rotate(x, qw, dim, eps_f, c.data(), s.data(), y.data());
        for (int64_t i = 0; i < dim; ++i) x[i] = static_cast<at::BFloat16>(y[i]);
      }
      if (slots[t] < 0 || slots[t] >= num_slots) continue;
      for (int64_t h = 0; h < kv_heads; ++h) {
        const int64_t row = slots[t] * kv_heads + h;
        rotate(kp + t * k.stride(0) + h * dim, kw, dim, eps_f, c.data(), s.data(), y.data());
        quantise(y.data(), dim, kc + row * dim, ks + row);
        const at::BFloat16* x = vp + t * v.stride(0) + h * dim;
        for (int64_t i = 0; i < dim; ++i) y[i] = static_cast<float>(x[i]);
        quantise(y.data(), dim, vc + row * dim, vs + row);
      }
    }
  });
  return std::count_if(slots, slots + tokens, [&](int64_t slot) { return slot >= num_slots; });
}

void check_pages(const char* op, const at::Tensor& k_scale, const at::Tensor& v_scale,
                 const at::Tensor& block_tables, const at::Tensor& seq_lens) {
  const int64_t blocks = k_scale.size(0), bs = k_scale.size(1), kv_heads = k_scale.size(2);
  const int64_t width = block_tables.size(1);
  const auto* tables = block_tables.const_data_ptr<int32_t>();
  const auto* seq = seq_lens.const_data_ptr<int32_t>();
  for (int64_t s = 0; s < seq_lens.numel(); ++s) {
    TORCH_CHECK(seq[s] >= 0 && seq[s] <= width * bs, op, ": request ", s, " of length ", seq[s],
                " does not fit a table of ", width, " blocks of ", bs);
    for (int64_t p = 0; p * bs < seq[s]; ++p) {
      const int64_t block = tables[s * width + p];
      TORCH_CHECK(block >= 0 && block < blocks, op, ": block ", block, " of request ", s,
                  " outside the cache of ", blocks);
      const int64_t count = std::min(bs, seq[s] - p * bs) * kv_heads;
      for (const at::Tensor* scale : {&k_scale, &v_scale}) {
        const auto* e = static_cast<const uint8_t*>(scale->const_data_ptr()) + block * bs * kv_heads;
        for (int64_t i = 0; i < count; ++i) {
          TORCH_CHECK(e[i] >= kScaleMin + kScaleBias && e[i] <= kScaleMax + kScaleBias, op,
                      ": a scale of 2^", int{e[i]} - kScaleBias, " in block ", block,
                      ", outside [2^", kScaleMin, ", 2^", kScaleMax, "]");
        }
      }
    }
  }
}

void cache_read_fp8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                    const at::Tensor& v_cache, const at::Tensor& k_scale,
                    const at::Tensor& v_scale, const at::Tensor& block_tables,
                    const at::Tensor& seq_lens) {
  check_pages("cache_read_fp8", k_scale, v_scale, block_tables, seq_lens);
  const int64_t bs = k_cache.size(1), kv_heads = k_cache.size(2), dim = k_cache.size(3);
  const int64_t width = block_tables.size(1), rows = width * bs;
  const auto* tables = block_tables.const_data_ptr<int32_t>();
  const auto* seq = seq_lens.const_data_ptr<int32_t>();
  const struct {
    at::BFloat16* out;
    const Code* codes;
    const uint8_t* scale;
  } sides[] = {{k.mutable_data_ptr<at::BFloat16>(), static_cast<const Code*>(k_cache.const_data_ptr()),
                static_cast<const uint8_t*>(k_scale.const_data_ptr())},
               {v.mutable_data_ptr<at::BFloat16>(), static_cast<const Code*>(v_cache.const_data_ptr()),
                static_cast<const uint8_t*>(v_scale.const_data_ptr())}};
  at::parallel_for(0, seq_lens.numel() * rows, 16, [&](int64_t begin, int64_t end) {
    for (int64_t r = begin; r < end; ++r) {
      const int64_t s = r / rows, j = r % rows;
      for (const auto& side : sides) {
        at::BFloat16* out = side.out + r * kv_heads * dim;
        if (j >= seq[s]) {
          std::fill(out, out + kv_heads * dim, at::BFloat16(0.0f));
          continue;
        }
        const int64_t slot = int64_t{tables[s * width + j / bs]} * bs + j % bs;
        for (int64_t h = 0; h < kv_heads; ++h) {
          const float f = scale_value(side.scale[slot * kv_heads + h]);
          const Code* codes = side.codes + (slot * kv_heads + h) * dim;
          for (int64_t d = 0; d < dim; ++d) {
            out[h * dim + d] = static_cast<at::BFloat16>(static_cast<float>(codes[d]) * f);
          }
        }
      }
    }
  });
}

void decode_attention_fp8(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& k_scale,
                          const at::Tensor& v_scale, const at::Tensor& block_tables,
                          const at::Tensor& seq_lens, double scale) {
  check_pages("decode_attention_fp8", k_scale, v_scale, block_tables, seq_lens);
  const int64_t requests = q.size(0), heads = q.size(1), dim = q.size(2);
  const int64_t bs = k_cache.size(1), kv_heads = k_cache.size(2), width = block_tables.size(1);
  const auto* tables = block_tables.const_data_ptr<int32_t>();
  const auto* seq = seq_lens.const_data_ptr<int32_t>();
  const auto* qp = q.const_data_ptr<at::BFloat16>();
  const auto* kc = static_cast<const Code*>(k_cache.const_data_ptr());
  const auto* vc = static_cast<const Code*>(v_cache.const_data_ptr());
  const auto* ks = static_cast<const uint8_t*>(k_scale.const_data_ptr());
  const auto* vs = static_cast<const uint8_t*>(v_scale.const_data_ptr());
  auto* op = out.mutable_data_ptr<at::BFloat16>();
  at::parallel_for(0, requests * heads, 1, [&](int64_t begin, int64_t end) {
    std::vector<float> x, sum(dim);
    for (int64_t u = begin; u < end; ++u) {
      const int64_t s = u / heads, h = u % heads, kh = h / (heads / kv_heads);
      const at::BFloat16* query = qp + s * q.stride(0) + h * dim;
      const auto row_of = [&](int64_t j) {
        return (int64_t{tables[s * width + j / bs]} * bs + j % bs) * kv_heads + kh;
      };
      x.resize(seq[s]);
      float top = -std::numeric_limits<float>::infinity();
      for (int64_t j = 0; j < seq[s]; ++j) {
        const int64_t row = row_of(j);
        double dot = 0.0;  // the largest queries times codes leave fp32, whatever the scale
        for (int64_t d = 0; d < dim; ++d) {
          dot += static_cast<double>(query[d]) * static_cast<double>(kc[row * dim + d]);
        }
        x[j] = static_cast<float>(dot * scale * scale_value(ks[row]));
        top = std::max(top, x[j]);
      }
      if (std::isinf(top) && top < 0) top = 0.0f;  // every score -infinity, or no row at all
      float total = 0.0f;
      std::fill(sum.begin(), sum.end(), 0.0f);
      for (int64_t j = 0; j < seq[s]; ++j) {
        const int64_t row = row_of(j);
        const float p = std::exp(x[j] - top), w = p * scale_value(vs[row]);
        total += p;
        for (int64_t d = 0; d < dim; ++d) sum[d] += w * static_cast<float>(vc[row * dim + d]);
      }
      for (int64_t d = 0; d < dim; ++d) {
        op[u * dim + d] = static_cast<at::BFloat16>(total == 0.0f ? 0.0f : sum[d] / total);
      }
    }
  });
}

}  // namespace svllm::ops::cpu_impl
