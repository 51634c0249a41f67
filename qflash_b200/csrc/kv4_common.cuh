// Shared by the kernels of the 4-bit key/value cache: its layout, the stored
// parameters and the element types at the boundary.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qflash_b200.h"
#include "qfb_internal.h"

namespace qfb {
namespace kv4 {

// A cache's buffers, all contiguous:
//   codes  [Z, H, C, D / 2] bytes, element 2i of a vector in the low half of byte i
//   param  [Z, H, C, 2] bf16: scale, zero point (a whole number 0..15)
//   weight [Z, H, C] fp32, lens [Z] int32, ctl [2] int32 (ticket, status)
struct Cache {
  uint8_t* codes[2];    // keys, values
  uint32_t* param[2];   // one 32-bit word per vector: scale in the low half, zero point in the high half
  float* weight;
  int32_t* lens;
  int32_t* ctl;
  int Z, H, C, D;
};

inline Cache view(const qflash_kv4_cache* c) {
  return {{(uint8_t*)c->k_codes, (uint8_t*)c->v_codes}, {(uint32_t*)c->k_param, (uint32_t*)c->v_param},
          c->weight, c->lens, c->ctl, c->Z, c->H, c->capacity, c->D};
}

__device__ __forceinline__ float param_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float param_zero(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Stored tokens of sequence z, whatever the buffer holds: never outside [0, C].
__device__ __forceinline__ int length_of(const Cache& c, int z) { return min(max(c.lens[z], 0), c.C); }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 8 fp32 numbers from a 16-byte boundary.  Plain loads, not the read-only path: what a kernel launched by
// launch_behind reads of the one before it is still being written when it begins.
__device__ __forceinline__ void read8(const float* p, float (&x)[8]) {  // on a 16-byte boundary
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
// 8 elements of one thread, as one or two 16-byte transfers where `vec` says
// that every row starts on a 16-byte boundary, else one by one.
template <class T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8]) {
  alignas(16) T r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = from_float<T>(x[i]);
  if (vec) {
    const uint4* w = reinterpret_cast<const uint4*>(r);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = r[i];
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// CTA `rank`'s copy of a word of shared memory
__device__ __forceinline__ uint32_t peer_word(const uint32_t* p, uint32_t rank) {
  uint32_t at, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// A kernel that begins while the one before it in the stream still runs: what it does before
// wait_for_previous may read nothing that one writes.  The one before says may_begin
// once all its CTAs are resident, so the second kernel's blocks take no place from it.
__device__ __forceinline__ void may_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class A>
inline void launch_behind(void (*kernel)(A), dim3 grid, unsigned threads, cudaStream_t s, const A& args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args);
}

int check_cache(const qflash_kv4_cache* c, const char* what);
int check_launch(const char* what, unsigned grid);

// See qflash_kv4_attend.
struct AttendArgs {
  Cache c;
  const void* q;
  void* out;
  int64_t qs[3], os[3];  // strides of (sequence, head, token) in elements
  int rep, N;            // query heads per key/value head, rows of the query tensor
  const int32_t* new_lens;
  int causal;
  float scale_log2e;
  const float* weights_in;  // null: no weights are accumulated
};

// Set into the mantissa of 128 (bf16) or 1024 (fp16), a code is a number.
constexpr uint32_t kMagicBf16 = 0x43004300u, kMagicFp16 = 0x64006400u;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

// What a unit of so many key tiles counts for where the attention kernels split their work: its queries
// and its output take the time of kBegin tiles.
constexpr int kBegin = 2;
__device__ __forceinline__ int cost_of(int tiles) { return tiles ? tiles + kBegin : 0; }

constexpr int kDevices = 64;  // as many as select_device knows

// Rows (tokens x rep) up to which the kernel for few rows also adds up weights.
constexpr int kWeightRows = 48;

// The rows of one sequence, and how many stored tokens they see at most.
struct Span {
  int len, fresh;  // stored tokens; rows of the query tensor that the sequence brings
  __device__ __forceinline__ int limit(const AttendArgs& a, int i) const {  // positions that token i sees
    return i >= fresh ? 0 : a.causal ? max(0, len - fresh + i + 1) : len;
  }
  __device__ __forceinline__ int most(const AttendArgs& a) const {
    return fresh ? limit(a, fresh - 1) : 0;
  }
};
__device__ __forceinline__ Span span_of(const AttendArgs& a, int z) {
  return {length_of(a.c, z), a.new_lens ? min(max(a.new_lens[z], 0), a.N) : a.N};
}

size_t rows_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights);
int attend_rows(const AttendArgs& a, bool fp16, void* ws, int dev, cudaStream_t s);
size_t prompt_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights);
int attend_prompt(const AttendArgs& a, bool fp16, void* ws, int dev, cudaStream_t s);

}  // namespace kv4
}  // namespace qfb
