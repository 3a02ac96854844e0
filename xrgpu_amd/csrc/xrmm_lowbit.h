// Microscaled 4-bit products (MX4) and the 8-bit paged cache: argument blocks of the
// launches, and the device helpers their kernels share.
#pragma once
#include "xrmm_device.h"

namespace xrmm {

// Storage types of the operators here (activations, outputs).
enum LT { LT_F32 = 0, LT_F16 = 1, LT_BF16 = 2 };

typedef __bf16 bf16;
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int MX_BLOCK = 32;  // values per scale
constexpr int MX_BLOB = 16;   // bytes of codes per block

struct MxQuantArgs {
  const void* x;
  uint8_t* codes;   // [rows, kb, 16]
  uint8_t* scales;  // [rows, kb]
  int64_t rows, K, kb;
  int dtype;        // LT
};

// Y [M, N] = A [M, K] W^T (+ bias); W as codes [N, kb, 16] and scales [N, kb].
struct MxArgs {
  const void* A;
  const uint8_t* As;  // A's scales [M, kb] when A holds MX4 codes, else null
  const uint8_t* B;
  const uint8_t* S;
  const void* bias;   // [N] of the output's type, or null
  void* Y;
  void* ws;           // split-K: arrival counters and float32 partials, or null
  int64_t ws_bytes;
  int64_t M, K, N, kb;
  int a_type;         // LT_F16 / LT_BF16 (As null), or -1 for MX4 codes
  int out;            // LT
};

// A paged cache: pages [P, Hkv, page, D] of 8-bit codes (int8, or e4m3 when fp8), one float32 scale for
// each page and head; token t of sequence b lies in page
// table[b, t / page], slot t % page.
struct KvCache {
  uint8_t *k, *v;
  float *ks, *vs;
  const int32_t* table;    // [B, width]
  const int32_t* lengths;  // [B]: tokens in the cache, the call's own among them
  const int32_t* starts;   // [B + 1]: each sequence's rows of the call, or null: `each` rows a sequence
  uint32_t* status;        // raised to 55 where a page or position does not exist; or null
  int64_t pages, rows;     // pages of the cache; rows (new tokens) of the call's own tensors
  int32_t B, each, width, Hkv, D, page, page_log2;
  bool fp8;
};

struct KvAppendArgs {
  KvCache c;
  const void *k, *v;           // [T, Hkv, D], token strides in elements
  int64_t k_stride, v_stride;
  int32_t max_new;
  int dtype;                   // LT
};

struct KvAttnArgs {
  KvCache c;
  const void* q;               // [T, Hq, D], token stride in elements
  void* o;                     // [T, Hq, D] contiguous
  void* ws;
  int64_t q_stride, ws_bytes;
  int32_t Hq, max_new, causal, window;
  float scale;
  int dtype;                   // LT_F16 / LT_BF16
  const int32_t* shared;       // pages of every sequence's first tokens (kv8_shared_attention), else null
  int32_t shared_pages;
  int32_t parts, part0;        // parts of a row in the workspace, and the first of a launch's own
  int64_t parts_at;            // where they begin
};

// A launch's threads along x are counted in 32 bits; a grid of more runs in part, without an error.
inline bool grid_counts(int64_t workgroups, int64_t threads) { return workgroups <= 0xFFFFFFFFll / threads; }

hipError_t launch_kv8_append(const KvAppendArgs& a, hipStream_t st);
hipError_t launch_kv8_attention(const KvAttnArgs& a, hipStream_t st);
int64_t kv8_workspace_bytes(const KvAttnArgs& a);
const char* kv8_kernel_name(const KvAttnArgs& a);
hipError_t launch_kv8_shared_attention(const KvAttnArgs& a, hipStream_t st);
int64_t kv8_shared_workspace_bytes(const KvAttnArgs& a);
const char* kv8_shared_kernel_name(const KvAttnArgs& a);

hipError_t launch_mx4_quantize(const MxQuantArgs& a, hipStream_t st);
hipError_t launch_matmul_mx4(const MxArgs& a, hipStream_t st);
int64_t mx4_workspace_bytes(int64_t M, int64_t K, int64_t N, int a_type);
const char* mx4_kernel_name(const MxArgs& a);

// The E8M0 scale 2^(byte - 127) as float32: byte 0 is the subnormal 2^-127, byte 255 NaN.
__device__ __forceinline__ float e8m0(uint32_t byte) {
  const uint32_t bits = byte == 0u ? 0x00400000u : byte == 255u ? 0x7FC00000u : byte << 23;
  return __builtin_bit_cast(float, bits);
}

// One output value in its storage type, rounded once (to nearest, ties to even).
__device__ __forceinline__ void st_lt(void* p, int64_t i, float v, int t) {
  if (t == LT_F32) static_cast<float*>(p)[i] = v;
  else if (t == LT_F16) static_cast<f16*>(p)[i] = static_cast<f16>(v);
  else static_cast<bf16*>(p)[i] = static_cast<bf16>(v);
}

__device__ __forceinline__ float ld_lt(const void* p, int64_t i, int t) {
  return t == LT_F32 ? static_cast<const float*>(p)[i]
         : t == LT_F16 ? static_cast<float>(static_cast<const f16*>(p)[i])
                       : static_cast<float>(static_cast<const bf16*>(p)[i]);
}

// Rows of sequence b in the call's own tensors: [first, first + count), count <= most. False, with no
// rows, where `starts` names others or more than the call was planned for.
__device__ __forceinline__ bool kv_rows(const KvCache& c, int b, int most, int& first, int& count) {
  if (c.starts == nullptr) {
    first = b * c.each;
    count = c.each;
    return true;
  }
  const int64_t f = c.starts[b], n = c.starts[b + 1] - f;
  const bool ok = f >= 0 && n >= 0 && n <= most && f + n <= c.rows;
  first = ok ? static_cast<int>(f) : 0;
  count = ok ? static_cast<int>(n) : 0;
  return ok;
}

// The page that holds token t of sequence b, or -1 where there is none: also past 2^31, where walks look ahead, as tables
// span less. Reads the table in any case (the host gives an empty one the address of the lengths), so that lookups need no branches.
__device__ __forceinline__ int32_t kv_page(const KvCache& c, int b, uint32_t t) {
  const uint32_t i = t >> c.page_log2;
  const bool in = i < static_cast<uint32_t>(c.width);
  const int32_t p = c.table[static_cast<int64_t>(b) * c.width + (in ? i : 0)];
  return in && p >= 0 && p < c.pages ? p : -1;
}

constexpr uint32_t KV_BAD = 55u;  // the status code of a row that names what does not exist

}  // namespace xrmm
