// extern "C" entry points of the serving operators (declarations in include/attnrank_b200.h): every
// argument is checked on the host before any device work.
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/attnrank_b200.h"
#include "capi_guard.h"
#include "layer_kernels.h"
#include "paged.h"

namespace {

constexpr double kTwoPi = 6.283185307179586476925286766559;

void require(bool ok, const char* who, const char* what) {
  if (!ok) throw arb::Error(std::string(who) + ": " + what);
}

bool aligned16(const void* pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 15) == 0; }
bool aligned4(const void* pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 3) == 0; }

void check_status_word(const char* who, const int* device_status) {
  require(aligned4(device_status), who, "device_status must be 4-byte aligned");
}

// Do any two of the rows [t * token_stride + h * head_stride, .. + head_dim), t < tokens, h < heads, share
// an element? Both strides are at least head_dim where there is more than one row along them.
bool rows_overlap(int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t head_dim) {
  using Wide = __int128;
  if (tokens == 1 || heads == 1 || Wide(heads - 1) * head_stride + head_dim <= token_stride ||
      Wide(tokens - 1) * token_stride + head_dim <= head_stride) {
    return false;  // the usual layouts: heads inside a token, or tokens inside a head
  }
  for (int64_t h = 1; h < heads; ++h) {  // rows h heads apart: the nearest multiples of token_stride
    const Wide apart = Wide(h) * head_stride;
    const Wide below = std::min<Wide>(apart / token_stride, tokens - 1);
    const Wide above = std::min<Wide>(below + 1, tokens - 1);
    if (apart - below * token_stride < head_dim) return true;
    if (above * token_stride - apart < head_dim && apart - above * token_stride < head_dim) return true;
  }
  return false;
}

// Makes the device that holds `array` current for the call, so that a call on another device's
// arrays and stream runs there. Asking the stream instead is not allowed while it is captured.
class ArrayDevice {
 public:
  explicit ArrayDevice(const void* array) {
    static const int devices = [] {
      int count = 0;
      return cudaGetDeviceCount(&count) == cudaSuccess ? count : 0;
    }();
    if (devices < 2) return;
    cudaPointerAttributes attributes{};
    int current = 0;
    arb::check_cuda(cudaPointerGetAttributes(&attributes, array), "array device");
    arb::check_cuda(cudaGetDevice(&current), "cudaGetDevice");
    if (attributes.type == cudaMemoryTypeDevice && attributes.device != current) {
      arb::check_cuda(cudaSetDevice(attributes.device), "cudaSetDevice");
      previous_ = current;
    }
  }
  ~ArrayDevice() {
    if (previous_ >= 0) cudaSetDevice(previous_);
  }
  ArrayDevice(const ArrayDevice&) = delete;
  ArrayDevice& operator=(const ArrayDevice&) = delete;

 private:
  int previous_ = -1;
};

// The scaled frequencies, radians a position, and the multiplier of cos and sin.
double scaled_frequencies(const char* who, const ar_rope_scaling& r, double* f) {
  require(r.rotary_dim >= 2 && r.rotary_dim <= 2 * arb::kMaxTableFrequencies && r.rotary_dim % 2 == 0, who,
          "rotary_dim must be even, 2..512");
  require(std::isfinite(r.theta) && r.theta > 1.0f, who, "theta must be finite and above 1");
  require(r.kind >= AR_ROPE_NONE && r.kind <= AR_ROPE_YARN, who, "unknown scaling kind");
  require(std::isfinite(r.attention_factor) && r.attention_factor >= 0.0f, who,
          "attention_factor must be finite and not negative");
  const bool windowed = r.kind == AR_ROPE_BANDS || r.kind == AR_ROPE_YARN;
  if (r.kind != AR_ROPE_NONE) {
    require(std::isfinite(r.factor) && r.factor >= 1.0f, who, "factor must be finite and at least 1");
  }
  if (windowed) {
    require(r.original_positions >= 1, who, "original_positions must be positive");
    require(std::isfinite(r.high) && r.low > 0.0f && r.high > r.low, who, "low and high must satisfy 0 < low < high");
  }
  const double log_theta = std::log(static_cast<double>(r.theta));
  const double factor = r.factor, low = r.low, high = r.high, window = r.original_positions;
  double ramp_begin = 0.0, ramp_length = 1.0;
  if (r.kind == AR_ROPE_YARN) {
    // the pair index at which `turns` rotations fit the window
    auto index = [&](double turns) { return r.rotary_dim * std::log(window / (kTwoPi * turns)) / (2.0 * log_theta); };
    ramp_begin = std::max(std::floor(index(high)), 0.0);
    ramp_length = std::max(std::min(std::ceil(index(low)), r.rotary_dim - 1.0) - ramp_begin, 0.001);
  }
  for (int i = 0; i < r.rotary_dim / 2; ++i) {
    const double base = std::exp(-2.0 * i / r.rotary_dim * log_theta);
    double slow = 0.0;  // share of the frequency that is divided by the factor
    if (r.kind == AR_ROPE_LINEAR) slow = 1.0;
    if (r.kind == AR_ROPE_BANDS) slow = 1.0 - std::min(std::max((window * base / kTwoPi - low) / (high - low), 0.0), 1.0);
    if (r.kind == AR_ROPE_YARN) slow = std::min(std::max((i - ramp_begin) / ramp_length, 0.0), 1.0);
    f[i] = r.kind == AR_ROPE_NONE ? base : slow * base / factor + (1.0 - slow) * base;
  }
  if (r.attention_factor != 0.0f) return r.attention_factor;
  return r.kind == AR_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
}

arb::PagedCache checked_cache(const char* who, const ar_paged_cache* cache) {
  require(cache != nullptr, who, "null cache");
  require(cache->dtype == AR_DTYPE_F16 || cache->dtype == AR_DTYPE_BF16, who, "dtype must be fp16 or bf16");
  require(cache->head_dim == 64 || cache->head_dim == 128, who, "head_dim must be 64 or 128");
  require(cache->page_size >= 16 && cache->page_size <= 1024 && (cache->page_size & (cache->page_size - 1)) == 0, who,
          "page_size must be a power of two, 16..1024");
  require(cache->kv_heads > 0 && cache->page_count > 0, who, "kv_heads and page_count must be positive");
  require(static_cast<int64_t>(cache->page_count) * cache->kv_heads <= INT32_MAX / cache->page_size, who,
          "the pool must hold fewer than 2^31 rows");
  require(cache->k_pages != nullptr && cache->v_pages != nullptr && aligned16(cache->k_pages) &&
              aligned16(cache->v_pages),
          who, "k_pages and v_pages must be 16-byte aligned device arrays");
  arb::PagedCache out;
  out.k_pages = cache->k_pages;
  out.v_pages = cache->v_pages;
  out.page_count = cache->page_count;
  while ((1 << out.page_shift) < cache->page_size) ++out.page_shift;
  out.kv_heads = cache->kv_heads;
  out.head_dim = cache->head_dim;
  out.dtype = cache->dtype;
  return out;
}

arb::PagedBatch checked_batch(const char* who, const ar_paged_batch* batch, const arb::PagedCache& cache) {
  require(batch != nullptr, who, "null batch");
  require(batch->sequence_count >= 0 && batch->token_count >= 0, who,
          "sequence_count and token_count must not be negative");
  require(batch->sequence_count <= 1 << 30, who, "sequence_count must be at most 2^30");
  require(batch->max_query_tokens > 0, who, "max_query_tokens must be positive");
  require(batch->page_table_stride > 0, who, "page_table_stride must be positive");
  if (batch->sequence_count > 0) {
    require(batch->q_offsets != nullptr && batch->kv_lengths != nullptr && batch->page_table != nullptr, who,
            "null batch array");
    require(aligned4(batch->q_offsets) && aligned4(batch->kv_lengths) && aligned4(batch->page_table), who,
            "q_offsets, kv_lengths and page_table must be 4-byte aligned");
  }
  arb::PagedBatch out;
  out.sequences = batch->sequence_count;
  out.tokens = batch->token_count;
  out.max_query = std::min(batch->max_query_tokens, std::max(batch->token_count, 1));
  out.table_stride = batch->page_table_stride;
  const int64_t capacity = static_cast<int64_t>(batch->page_table_stride) << cache.page_shift;
  out.capacity = static_cast<int>(std::min<int64_t>(capacity, INT32_MAX - 1024));  // tile ends stay below 2^31
  out.q_offsets = batch->q_offsets;
  out.kv_lengths = batch->kv_lengths;
  out.page_table = batch->page_table;
  return out;
}

void check_query_heads(const char* who, int query_heads, const arb::PagedCache& cache) {
  require(query_heads > 0 && query_heads % cache.kv_heads == 0 && query_heads / cache.kv_heads <= 128, who,
          "query_heads must be a positive multiple of kv_heads, at most 128 times it");
}

int attention_call(const char* who, const ar_paged_cache* cache, const ar_paged_batch* batch, const void* q,
                   int64_t q_stride, int query_heads, float scale, int sliding_window, void* out, int64_t out_stride,
                   float* lse, void* workspace, int64_t workspace_bytes, int* device_status, void* stream,
                   uint32_t self_test_blocks) {
  arb::PagedAttentionArgs args;
  args.cache = checked_cache(who, cache);
  args.batch = checked_batch(who, batch, args.cache);
  check_query_heads(who, query_heads, args.cache);
  require(args.batch.max_query <= 1 << 24, who, "max_query_tokens must be at most 2^24");
  const int64_t width = static_cast<int64_t>(query_heads) * args.cache.head_dim;
  require(q_stride >= width && q_stride % 8 == 0 && out_stride >= width && out_stride % 8 == 0, who,
          "q_stride and out_stride must be multiples of 8 and hold the query heads");
  require(std::isfinite(scale) && scale >= 0.0f, who, "scale must be finite and not negative (0: 1/sqrt(head_dim))");
  const double chosen = scale != 0.0f ? scale : 1.0 / std::sqrt(static_cast<double>(args.cache.head_dim));
  args.scale_log2 = static_cast<float>(chosen * 1.4426950408889634074);
  require(std::isnormal(args.scale_log2), who, "scale times log2(e) must be a normal fp32 number");
  require(sliding_window >= 0, who, "sliding_window must not be negative");
  if (args.batch.tokens == 0 || args.batch.sequences == 0) return AR_OK;
  require(q != nullptr && out != nullptr && aligned16(q) && aligned16(out), who,
          "q and out must be 16-byte aligned device arrays");
  require(q != out, who, "out must not overlap q");
  require(aligned4(lse), who, "lse must be 4-byte aligned");
  check_status_word(who, device_status);
  const int64_t needed = arb::paged_attention_workspace(args.cache, args.batch, query_heads);
  if (needed > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < needed)) {
    throw arb::Error(std::string(who) + ": needs a 16-byte aligned workspace of " + std::to_string(needed) + " bytes");
  }
  args.q = q;
  args.q_stride = q_stride;
  args.query_heads = query_heads;
  args.sliding_window = sliding_window;
  args.out = out;
  args.out_stride = out_stride;
  args.lse = lse;
  args.workspace = workspace;
  args.status = device_status;
  args.self_test_blocks = self_test_blocks;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ArrayDevice device(cache->k_pages);
  arb::check_cuda(arb::launch_paged_attention(args, s), who);
  return AR_OK;
}

}  // namespace

extern "C" {

int ar_rope_frequencies(const ar_rope_scaling* scaling, double* frequencies_out, double* multiplier_out) {
  return arb::guarded_call([&] {
    const char* who = "rope_frequencies";
    require(scaling != nullptr && frequencies_out != nullptr, who, "null argument");
    const double multiplier = scaled_frequencies(who, *scaling, frequencies_out);
    if (multiplier_out != nullptr) *multiplier_out = multiplier;
    return AR_OK;
  });
}

int ar_rope_table_scaled(const ar_rope_scaling* scaling, int positions, float* cos_table, float* sin_table,
                         void* stream) {
  return arb::guarded_call([&] {
    const char* who = "rope_table_scaled";
    require(scaling != nullptr, who, "null argument");
    arb::TableTurns turns{};
    const double multiplier = scaled_frequencies(who, *scaling, turns.value);
    require(positions >= 0 && positions <= 1 << 30, who, "positions must be 0..2^30");
    if (positions == 0) return AR_OK;
    require(cos_table != nullptr && sin_table != nullptr && aligned16(cos_table) && aligned16(sin_table), who,
            "the tables must be 16-byte aligned device arrays");
    const int half = scaling->rotary_dim / 2;
    for (int i = 0; i < half; ++i) turns.value[i] /= kTwoPi;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ArrayDevice device(cos_table);
    arb::check_cuda(arb::launch_rope_table_scaled(turns, half, static_cast<float>(multiplier), positions, cos_table,
                                                  sin_table, s),
                    who);
    return AR_OK;
  });
}

int ar_rotary_positions(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* out,
                        int64_t out_token_stride, int64_t out_head_stride, const int32_t* positions, int token_count,
                        int heads, int head_dim, int rotary_dim, int interleaved, int inverse, const float* cos_table,
                        const float* sin_table, int table_positions, int* device_status, int dtype, void* stream) {
  return arb::guarded_call([&] {
    const char* who = "rotary_positions";
    require(dtype == AR_DTYPE_F16 || dtype == AR_DTYPE_BF16, who, "dtype must be fp16 or bf16");
    require(token_count >= 0 && heads >= 0 && table_positions >= 0, who, "counts must not be negative");
    require(heads <= 65536, who, "heads must be at most 65536");
    require(head_dim >= 2 && head_dim <= 1024, who, "head_dim must be 2..1024");
    require(rotary_dim >= 2 && rotary_dim <= head_dim && rotary_dim % 2 == 0, who,
            "rotary_dim must be even, 2..head_dim");
    if (token_count == 0 || heads == 0) return AR_OK;
    require(x != nullptr && out != nullptr && positions != nullptr && cos_table != nullptr && sin_table != nullptr, who,
            "null argument");
    require(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 1) == 0, who,
            "x and out must be aligned to their type");
    require(aligned4(positions) && aligned4(cos_table) && aligned4(sin_table), who,
            "positions and the tables must be 4-byte aligned");
    require(x_head_stride >= 0 && x_token_stride >= 0, who, "strides must not be negative");
    require((heads == 1 || out_head_stride >= head_dim) && (token_count == 1 || out_token_stride >= head_dim), who,
            "out's strides must be at least head_dim, or its rows would overlap");
    require(!rows_overlap(token_count, out_token_stride, heads, out_head_stride, head_dim), who,
            "out's strides would make its rows overlap");
    require(out != x || (out_token_stride == x_token_stride && out_head_stride == x_head_stride), who,
            "in place needs x's strides");
    check_status_word(who, device_status);
    arb::RotaryArgs args;
    args.x = x;
    args.x_token_stride = x_token_stride;
    args.x_head_stride = x_head_stride;
    args.out = out;
    args.out_token_stride = out_token_stride;
    args.out_head_stride = out_head_stride;
    args.positions = positions;
    args.tokens = token_count;
    args.heads = heads;
    args.head_dim = head_dim;
    args.rotary_dim = rotary_dim;
    args.interleaved = interleaved != 0;
    args.inverse = inverse != 0;
    args.cos_table = cos_table;
    args.sin_table = sin_table;
    args.table_positions = table_positions;
    args.status = device_status;
    args.dtype = dtype;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ArrayDevice device(out);
    arb::check_cuda(arb::launch_rotary_positions(args, s), who);
    return AR_OK;
  });
}

int ar_paged_append(const ar_paged_cache* cache, const ar_paged_batch* batch, const void* qkv, int64_t qkv_stride,
                    const float* bias, int query_heads, void* q_out, int64_t q_out_stride, const float* cos_table,
                    const float* sin_table, int table_positions, int rotary_dim, int interleaved, int* device_status,
                    void* stream) {
  return arb::guarded_call([&] {
    const char* who = "paged_append";
    arb::PagedAppendArgs args;
    args.cache = checked_cache(who, cache);
    args.batch = checked_batch(who, batch, args.cache);
    require(query_heads >= 0 && query_heads <= 65536 && args.cache.kv_heads <= 65536, who,
            "query_heads and kv_heads must be at most 65536, query_heads not negative");
    const int head_dim = args.cache.head_dim;
    const int64_t width = (static_cast<int64_t>(query_heads) + 2 * args.cache.kv_heads) * head_dim;
    require(qkv_stride >= width && qkv_stride % 8 == 0, who,
            "qkv_stride must be a multiple of 8 and hold the row's heads");
    require(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 16 == 0, who,
            "rotary_dim must be a multiple of 16, 0..head_dim");
    require(table_positions >= 0, who, "table_positions must not be negative");
    if (rotary_dim > 0) {
      require(cos_table != nullptr && sin_table != nullptr && aligned16(cos_table) && aligned16(sin_table), who,
              "the tables must be 16-byte aligned device arrays");
    }
    if (q_out != nullptr && query_heads > 0) {
      require(aligned16(q_out), who, "q_out must be 16-byte aligned");
      require(q_out_stride >= static_cast<int64_t>(query_heads) * head_dim && q_out_stride % 8 == 0, who,
              "q_out_stride must be a multiple of 8 and hold the query heads");
      require(q_out != qkv || q_out_stride == qkv_stride, who, "in place needs qkv's stride");
    }
    if (args.batch.tokens == 0 || args.batch.sequences == 0) return AR_OK;
    require(qkv != nullptr && aligned16(qkv), who, "qkv must be a 16-byte aligned device array");
    require(bias == nullptr || aligned16(bias), who, "bias must be 16-byte aligned");
    check_status_word(who, device_status);
    args.qkv = qkv;
    args.qkv_stride = qkv_stride;
    args.bias = bias;
    args.query_heads = query_heads;
    args.q_out = query_heads > 0 ? q_out : nullptr;
    args.q_out_stride = q_out_stride;
    args.cos_table = cos_table;
    args.sin_table = sin_table;
    args.table_positions = table_positions;
    args.rotary_dim = rotary_dim;
    args.interleaved = interleaved != 0;
    args.status = device_status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ArrayDevice device(cache->k_pages);
    arb::check_cuda(arb::launch_paged_append(args, s), who);
    return AR_OK;
  });
}

int64_t ar_paged_attention_workspace(const ar_paged_cache* cache, const ar_paged_batch* batch, int query_heads) {
  int64_t bytes = -1;
  arb::guarded_call([&] {
    const char* who = "paged_attention_workspace";
    const arb::PagedCache c = checked_cache(who, cache);
    const arb::PagedBatch b = checked_batch(who, batch, c);
    check_query_heads(who, query_heads, c);
    bytes = arb::paged_attention_workspace(c, b, query_heads);
    return AR_OK;
  });
  return bytes;
}

int ar_paged_attention(const ar_paged_cache* cache, const ar_paged_batch* batch, const void* q, int64_t q_stride,
                       int query_heads, float scale, int sliding_window, void* out, int64_t out_stride, float* lse,
                       void* workspace, int64_t workspace_bytes, int* device_status, void* stream) {
  return arb::guarded_call([&] {
    return attention_call("paged_attention", cache, batch, q, q_stride, query_heads, scale, sliding_window, out, out_stride,
                          lse, workspace, workspace_bytes, device_status, stream, ~0u);
  });
}

int ar_paged_attention_wait_selftest(const ar_paged_cache* cache, const ar_paged_batch* batch, const void* q,
                                     int64_t q_stride, int query_heads, int sliding_window, void* out, int64_t out_stride,
                                     float* lse, void* workspace, int64_t workspace_bytes, uint32_t blocks,
                                     int* device_status, void* stream) {
  return arb::guarded_call([&] {
    return attention_call("paged_attention_wait_selftest", cache, batch, q, q_stride, query_heads, 0.0f, sliding_window, out,
                          out_stride, lse, workspace, workspace_bytes, device_status, stream, blocks);
  });
}

}  // extern "C"
