// kv8.h -- the 8-bit paged cache (dsd_kv8_*): launch interface of
// kv8_append.hip, kv8_attend.hip and kv8_prompt.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "dsd_hip.h"
#include "dsd_internal.h"

namespace dsdk {

// A cache's memory (the layout in include/dsd_hip.h).
struct Kv8View {
  uint8_t* keys = nullptr;
  uint8_t* values = nullptr;
  float* key_scales = nullptr;
  float* value_scales = nullptr;
  float* summaries = nullptr;  // null: none kept
  int* token_counts = nullptr;
  int heads = 0;  // key heads
  int dim = 0;
  int page = 0;    // tokens
  int chunks = 0;  // page / 16
  int capacity = 0;
  int format = 0;  // DSD_KV8_*
};

struct Kv8Rotation {
  // [4][256][pairs]: (cos, sin) of pair p turned by j * 256^level positions
  const double2* table = nullptr;
  int pairs = 0;
  int interleaved = 0;
  double magnitude = 1.0;
};

struct Kv8AppendArgs {
  Kv8View c;
  Kv8Rotation rot;
  dsd_kv8_batch b = {};
  int type = 0;  // DSD_TYPE_*
  int q_heads = 0;
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  void* q_out = nullptr;
  int64_t q_stride = 0, k_stride = 0, v_stride = 0, out_stride = 0;  // elements
  FailReport fail;
};
void LaunchKv8Append(const Kv8AppendArgs& a, hipStream_t stream);

struct Kv8AttendArgs {
  Kv8View c;
  dsd_kv8_batch b = {};
  int type = 0;
  int q_heads = 0;
  bool causal = false;  // several query tokens a request, each over what precedes it
  const void* q = nullptr;
  void* out = nullptr;
  int64_t q_stride = 0, out_stride = 0;  // elements
  float scale = 0.0f;
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  FailReport fail;
};
void LaunchKv8Attend(const Kv8AttendArgs& a, hipStream_t stream);
// The form of it for many rows (kv8_prompt.hip).
void LaunchKv8Prompt(const Kv8AttendArgs& a, hipStream_t stream);
size_t Kv8PromptWorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads);
size_t Kv8WorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads);
// Each key head's queries summed, in order, in float32: sums[batch][heads * dim].
void LaunchKv8GroupQueries(const Kv8View& c, int batch, int type, int q_heads, const void* q,
                           int64_t q_stride, float* sums, hipStream_t stream);
// The kernels that calls on such a cache run.
void PreloadKv8Append(const Kv8View& c);
void PreloadKv8Attend(const Kv8View& c);
void PreloadKv8Prompt(const Kv8View& c);

}  // namespace dsdk
