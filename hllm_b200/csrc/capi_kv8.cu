// capi_kv8.cu -- C entry points of the 8-bit paged KV cache
// (include/hllm_b200.h): argument checks, then the launches of kv8_cache.cu and
// kv8_attention.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "hllm_b200.h"
#include "kv8.cuh"

namespace hb {
void set_last_error(const std::string& message);  // stage.cu
}

namespace {

hllm_b200_status refuse(const char* why) {
  try {
    hb::set_last_error(why);
  } catch (...) {  // no exception crosses the ABI
  }
  return HLLM_B200_INVALID_REQUEST;
}

hllm_b200_status cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return HLLM_B200_OK;
  try {
    hb::set_last_error(cudaGetErrorString(e));
  } catch (...) {
  }
  return e == cudaErrorInvalidValue ? HLLM_B200_INVALID_REQUEST : HLLM_B200_INTERNAL;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr uint64_t kMaxInt = 0x7fffffff;
// Keys of a row in attention: its passes count, in 32 bits, up to a few key tiles
// past the last one.
constexpr uint64_t kMostKeys = kMaxInt - 4096;

// The first fault of a cache description, or null.
const char* cache_fault(const hllm_b200_kv8* c) {
  if (!c) return "8-bit KV cache: null cache";
  if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales)
    return "8-bit KV cache: null array";
  if (!aligned16(c->k_codes) || !aligned16(c->k_scales) || !aligned16(c->v_codes) ||
      !aligned16(c->v_scales))
    return "8-bit KV cache: arrays must be 16-byte aligned";
  if (c->head_dim == 0 || c->head_dim % 32 != 0 || c->head_dim > hb::kKv8MaxDim)
    return "8-bit KV cache: head_dim must be a multiple of 32, at most 256";
  if (c->kv_heads == 0 || c->kv_heads > 65535) return "8-bit KV cache: bad kv_heads";
  if (c->blocks == 0 || c->blocks > kMaxInt / hb::kKv8Page ||
      c->blocks * c->kv_heads > kMaxInt)
    return "8-bit KV cache: blocks x 16 and blocks x kv_heads must be 1 to 2^31 - 1";
  return nullptr;
}

const char* heads_fault(uint32_t hq, uint32_t hkv) {
  if (hq == 0 || hq % hkv != 0 || hq > 65535)
    return "8-bit KV cache: query heads must be a multiple of kv_heads";
  return nullptr;
}

hb::Kv8Cache cache_of(const hllm_b200_kv8* c) {
  return hb::Kv8Cache{c->k_codes,
                      c->k_scales,
                      c->v_codes,
                      c->v_scales,
                      static_cast<long long>(c->blocks),
                      static_cast<int>(c->kv_heads),
                      static_cast<int>(c->head_dim)};
}

bool known_type(hllm_b200_dtype t) {
  return t == HLLM_B200_F32 || t == HLLM_B200_F16 || t == HLLM_B200_BF16;
}

cudaError_t current_sm_count(int* sm_count) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  return cudaDeviceGetAttribute(sm_count, cudaDevAttrMultiProcessorCount, dev);
}

}  // namespace

extern "C" {

hllm_b200_status hllm_b200_rope_turns(const hllm_b200_rope* rope, double* turns, float* factor) {
  if (!rope || !turns || !factor) return refuse("rope: null argument");
  const hllm_b200_rope& p = *rope;
  if (p.rotary_dim == 0 || p.rotary_dim % 2 != 0 || p.rotary_dim > hb::kKv8MaxDim)
    return refuse("rope: rotary_dim must be even, 2 to 256");
  if (!(std::isfinite(p.theta) && p.theta > 1.0)) return refuse("rope: theta must be above 1");
  if (!std::isfinite(p.attention_factor) || p.attention_factor < 0.0)
    return refuse("rope: bad attention_factor");
  if (p.scaling > HLLM_B200_ROPE_YARN) return refuse("rope: unknown scaling");
  if (p.scaling != HLLM_B200_ROPE_NONE && !(std::isfinite(p.factor) && p.factor >= 1.0))
    return refuse("rope: the scaling factor must be at least 1");
  const bool by_length = p.scaling == HLLM_B200_ROPE_LLAMA3 || p.scaling == HLLM_B200_ROPE_YARN;
  if (by_length && !(std::isfinite(p.original_max_position) && p.original_max_position > 0.0))
    return refuse("rope: original_max_position must be positive");
  if (p.scaling == HLLM_B200_ROPE_LLAMA3 &&
      !(p.low_freq_factor > 0.0 && p.high_freq_factor > p.low_freq_factor &&
        std::isfinite(p.high_freq_factor)))
    return refuse("rope: 0 < low_freq_factor < high_freq_factor is needed");
  if (p.scaling == HLLM_B200_ROPE_YARN &&
      !(p.beta_slow > 0.0 && p.beta_fast > p.beta_slow && std::isfinite(p.beta_fast)))
    return refuse("rope: beta_fast > beta_slow > 0 is needed");
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  const double n = p.rotary_dim;
  double low = 0.0, high = 0.0;
  if (p.scaling == HLLM_B200_ROPE_YARN) {
    // The pair that turns b times within the original length:
    // theta^(-2i/n) * length / (2 pi) = b.
    auto pair_of = [&](double b) {
      return n * std::log(p.original_max_position / (b * kTwoPi)) / (2.0 * std::log(p.theta));
    };
    low = std::fmax(std::floor(pair_of(p.beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(p.beta_slow)), n - 1.0);
  }
  for (uint32_t i = 0; i < p.rotary_dim / 2; ++i) {
    double f = std::pow(p.theta, -2.0 * i / n);
    if (p.scaling == HLLM_B200_ROPE_LINEAR) {
      f /= p.factor;
    } else if (p.scaling == HLLM_B200_ROPE_LLAMA3) {
      const double wave = kTwoPi / f, old = p.original_max_position;
      if (wave > old / p.low_freq_factor) {
        f /= p.factor;
      } else if (wave >= old / p.high_freq_factor) {
        const double mix =
            (old / wave - p.low_freq_factor) / (p.high_freq_factor - p.low_freq_factor);
        f = (1.0 - mix) * f / p.factor + mix * f;
      }
    } else if (p.scaling == HLLM_B200_ROPE_YARN) {
      const double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 0.001), 0.0), 1.0);
      f = f / p.factor * ramp + f * (1.0 - ramp);
    }
    turns[i] = f / kTwoPi;
  }
  *factor = static_cast<float>(p.attention_factor > 0.0 ? p.attention_factor
                               : p.scaling == HLLM_B200_ROPE_YARN
                                   ? 0.1 * std::log(p.factor) + 1.0
                                   : 1.0);
  return HLLM_B200_OK;
}

hllm_b200_status hllm_b200_kv8_write(const hllm_b200_kv8* cache, const void* qkv,
                                     hllm_b200_dtype dtype, uint64_t tokens, uint32_t hq,
                                     const int32_t* positions, const int32_t* slots,
                                     const float* q_norm, const float* k_norm, float eps,
                                     const double* turns, uint32_t rotary_dim,
                                     uint32_t interleaved, float factor, uint16_t* q_out,
                                     uint32_t* status, void* stream) {
  if (const char* why = cache_fault(cache)) return refuse(why);
  if (const char* why = heads_fault(hq, cache->kv_heads)) return refuse(why);
  if (!known_type(dtype)) return refuse("8-bit KV write: qkv must be F32, F16 or BF16");
  if (tokens > kMaxInt) return refuse("8-bit KV write: too many tokens");
  if (rotary_dim % 2 != 0 || rotary_dim > cache->head_dim)
    return refuse("8-bit KV write: rotary_dim must be even and at most head_dim");
  if (!std::isfinite(eps) || eps < 0.f) return refuse("8-bit KV write: bad eps");
  if (!std::isfinite(factor)) return refuse("8-bit KV write: bad factor");
  if (!status) return refuse("8-bit KV write: null status");
  if (tokens == 0) return HLLM_B200_OK;
  if (!qkv || !positions || !slots || !q_out || (rotary_dim && !turns))
    return refuse("8-bit KV write: null argument");
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm))
    return refuse("8-bit KV write: qkv, q_out and norm weights must be 16-byte aligned");
  hb::Kv8WriteArgs a{};
  a.cache = cache_of(cache);
  a.qkv = qkv;
  a.type = static_cast<int>(dtype);
  a.tokens = static_cast<int>(tokens);
  a.hq = static_cast<int>(hq);
  a.positions = positions;
  a.slots = slots;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.turns = turns;
  a.rotary = static_cast<int>(rotary_dim);
  a.interleaved = interleaved ? 1 : 0;
  a.factor = factor;
  a.q_out = reinterpret_cast<__half*>(q_out);
  a.status = status;
  return cuda_status(hb::kv8_write_launch(a, static_cast<cudaStream_t>(stream)));
}

hllm_b200_status hllm_b200_kv8_read(const hllm_b200_kv8* cache, const int32_t* block_tables,
                                    uint32_t rows, uint32_t max_blocks, const int32_t* first,
                                    const int32_t* lengths, const int32_t* offsets,
                                    uint64_t tokens, hllm_b200_dtype dtype, void* k_out,
                                    void* v_out, uint32_t* status, void* stream) {
  if (const char* why = cache_fault(cache)) return refuse(why);
  if (!known_type(dtype)) return refuse("8-bit KV read: the output must be F32, F16 or BF16");
  if (tokens > kMaxInt - 64) return refuse("8-bit KV read: too many tokens");
  if (rows > kMaxInt / 2 || max_blocks > kMaxInt / hb::kKv8Page)
    return refuse("8-bit KV read: rows or max_blocks out of range");
  if (!status) return refuse("8-bit KV read: null status");
  if (tokens == 0 || rows == 0) return HLLM_B200_OK;
  if (max_blocks == 0 || !block_tables || !lengths || !offsets || !k_out || !v_out)
    return refuse("8-bit KV read: null argument");
  if (!aligned16(k_out) || !aligned16(v_out))
    return refuse("8-bit KV read: outputs must be 16-byte aligned");
  hb::Kv8ReadArgs a{};
  a.cache = cache_of(cache);
  a.tables = block_tables;
  a.first = first;
  a.lengths = lengths;
  a.offsets = offsets;
  a.rows = static_cast<int>(rows);
  a.max_blocks = static_cast<int>(max_blocks);
  a.tokens = static_cast<int>(tokens);
  a.type = static_cast<int>(dtype);
  a.k_out = k_out;
  a.v_out = v_out;
  a.status = status;
  return cuda_status(hb::kv8_read_launch(a, static_cast<cudaStream_t>(stream)));
}

hllm_b200_status hllm_b200_kv8_attention_workspace(uint32_t rows, uint64_t tokens,
                                                   uint64_t max_row_tokens, uint32_t hq,
                                                   uint32_t kv_heads, uint32_t head_dim,
                                                   uint64_t* bytes) {
  if (!bytes) return refuse("8-bit KV attention: null argument");
  if (kv_heads == 0 || kv_heads > 65535) return refuse("8-bit KV cache: bad kv_heads");
  if (const char* why = heads_fault(hq, kv_heads)) return refuse(why);
  if (head_dim == 0 || head_dim % 32 != 0 || head_dim > hb::kKv8MaxDim)
    return refuse("8-bit KV cache: head_dim must be a multiple of 32, at most 256");
  if (rows > kMaxInt / 2 || tokens > kMaxInt || max_row_tokens > kMaxInt)
    return refuse("8-bit KV attention: rows or tokens out of range");
  int sm_count = 0;
  const cudaError_t e = current_sm_count(&sm_count);
  if (e != cudaSuccess) return cuda_status(e);
  *bytes = hb::kv8_attention_workspace(static_cast<int>(max_row_tokens), static_cast<int>(hq),
                                       static_cast<int>(kv_heads), static_cast<int>(head_dim),
                                       sm_count);
  return HLLM_B200_OK;
}

hllm_b200_status hllm_b200_kv8_attention(const hllm_b200_kv8* cache, const uint16_t* q,
                                         uint64_t ld_q, const int32_t* cu_seqlens,
                                         const int32_t* lengths, const int32_t* block_tables,
                                         uint32_t rows, uint64_t tokens, uint64_t max_row_tokens,
                                         uint32_t hq, uint32_t max_blocks, float scale,
                                         uint16_t* out, uint64_t ld_out, void* workspace,
                                         uint64_t workspace_bytes, uint32_t* status, void* stream) {
  if (const char* why = cache_fault(cache)) return refuse(why);
  if (const char* why = heads_fault(hq, cache->kv_heads)) return refuse(why);
  if (rows > kMaxInt / 2 || tokens > kMaxInt || max_row_tokens > kMaxInt ||
      max_blocks > kMostKeys / hb::kKv8Page)
    return refuse("8-bit KV attention: rows, tokens or max_blocks out of range");
  if (!std::isfinite(scale)) return refuse("8-bit KV attention: bad scale");
  if (!status) return refuse("8-bit KV attention: null status");
  const uint64_t width = static_cast<uint64_t>(hq) * cache->head_dim;
  if (ld_q < width || ld_out < width || ld_q % 8 != 0 || ld_out % 8 != 0 || ld_q > kMaxInt ||
      ld_out > kMaxInt)
    return refuse("8-bit KV attention: row strides must be multiples of 8, at least Hq x d");
  if (rows == 0 || tokens == 0) return HLLM_B200_OK;
  if (max_blocks == 0 || max_row_tokens == 0 || !q || !cu_seqlens || !lengths || !block_tables ||
      !out || !workspace)
    return refuse("8-bit KV attention: null argument");
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace))
    return refuse("8-bit KV attention: q, out and workspace must be 16-byte aligned");
  int sm_count = 0;
  const cudaError_t e = current_sm_count(&sm_count);
  if (e != cudaSuccess) return cuda_status(e);
  hb::Kv8AttnArgs a{};
  a.cache = cache_of(cache);
  a.q = reinterpret_cast<const __half*>(q);
  a.ld_q = static_cast<long long>(ld_q);
  a.cu_seqlens = cu_seqlens;
  a.lengths = lengths;
  a.tables = block_tables;
  a.rows = static_cast<int>(rows);
  a.tokens = static_cast<int>(tokens);
  a.max_row_tokens = static_cast<int>(max_row_tokens);
  a.hq = static_cast<int>(hq);
  a.max_blocks = static_cast<int>(max_blocks);
  a.scale = scale;
  a.out = reinterpret_cast<__half*>(out);
  a.ld_out = static_cast<long long>(ld_out);
  a.workspace = static_cast<float*>(workspace);
  a.status = status;
  a.sm_count = sm_count;
  if (workspace_bytes <
      hb::kv8_attention_workspace(a.max_row_tokens, a.hq, a.cache.hkv, a.cache.dim, sm_count)) {
    refuse("8-bit KV attention: the workspace is too small");
    return HLLM_B200_RESOURCE_EXHAUSTED;
  }
  return cuda_status(hb::kv8_attention_launch(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
