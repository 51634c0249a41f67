// The 4-bit key/value cache: quantising new tokens into it, reading values out
// of it, packing what eviction keeps into another cache, and the C entry points.
//
// Quantisation of a vector x of D elements, every step rounded as said:
//   lo = min(x, 0), hi = max(x, 0)
//   scale = bf16(fp32((hi - lo) / 15)), the range and its division in fp64
//   zero  = clamp(rint(fp32(-lo / scale)), 0, 15)
//   code  = clamp(rint(fp32(x / scale)) + zero, 0, 15)
// rint to even.  A vector of zeros has scale 0; one with an infinity or a NaN
// has scale NaN (all it stands for is NaN) and codes 0.
#include <algorithm>

#include "kv4_common.cuh"

namespace qfb {
namespace kv4 {

int check_launch(const char* what, unsigned grid) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_err(QFLASH_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  note_launch((int)grid);
  return QFLASH_OK;
}

// ---------------------------------------------------------------- append
struct AppendArgs {
  Cache c;
  const void* x[2];
  int64_t st[2][3];
  int N;
  const int32_t* new_lens;
  const int32_t* at;
  bool vec[2];
};

constexpr int kThreads = 256;

// D / 8 lanes per vector, 8 elements each.
template <class T, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a) {
  constexpr int L = D / 8;
  const Cache& c = a.c;
  const int lane = threadIdx.x % L;
  const unsigned row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const unsigned n = row % a.N, rest = row / a.N, h = rest % c.H, kv = rest / c.H & 1, z = rest / c.H / 2;
  if (z < (unsigned)c.Z) {  // whole groups of L lanes leave together
    const int base = a.at ? a.at[z] : c.lens[z];
    const int fresh = a.new_lens ? min(max(a.new_lens[z], 0), a.N) : a.N;
    const long long pos = (long long)base + n;
    if ((int)n < fresh && pos >= 0 && pos < c.C) {
      float x[8];
      load8((const T*)a.x[kv] + z * a.st[kv][0] + h * a.st[kv][1] + n * a.st[kv][2] + lane * 8, a.vec[kv], x);
      float lo = 0.f, hi = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad |= !(fabsf(x[i]) < INFINITY);
      }
      const unsigned group = (L == 32 ? ~0u : (1u << L) - 1) << (threadIdx.x % 32 / L * L);
#pragma unroll
      for (int o = L / 2; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(group, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(group, hi, o));
      }
      bad = __any_sync(group, bad);
      __nv_bfloat16 scale = __float2bfloat16_rn((float)(((double)hi - (double)lo) / 15.0));
      if (bad) scale = __ushort_as_bfloat16(0x7fc0);
      const float s = __bfloat162float(scale);
      float zero = 0.f;
      uint32_t word = 0;
      if (s > 0.f) {
        zero = fminf(rintf(__fdiv_rn(-lo, s)), 15.f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x[i], s)) + zero, 0.f), 15.f) << (4 * i);
      }
      const size_t to = ((size_t)z * c.H + h) * c.C + pos;
      reinterpret_cast<uint32_t*>(c.codes[kv])[to * (D / 8) + lane] = word;
      if (lane == 0) {
        c.param[kv][to] = (uint32_t)__bfloat16_as_ushort(scale) | (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(zero)) << 16;
        if (kv == 0) c.weight[to] = 0.f;
      }
    }
  }
  // The last CTA moves lens on, after every CTA has read them.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&c.ctl[0], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int i = threadIdx.x; i < c.Z; i += kThreads) {
    const int base = a.at ? a.at[i] : c.lens[i];
    const long long end = (long long)base + (a.new_lens ? min(max(a.new_lens[i], 0), a.N) : a.N);
    if (base < 0 || end > c.C) atomicOr(&c.ctl[1], 1);
    c.lens[i] = (int)min(max(end, 0LL), (long long)c.C);
  }
  if (threadIdx.x == 0) c.ctl[0] = 0;
}

// ---------------------------------------------------------------- read
struct ReadArgs {
  Cache c;
  void* out[2];
  int N;
  const int32_t* start;
};

template <class T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs a) {
  constexpr int L = D / 8;
  const Cache& c = a.c;
  const int lane = threadIdx.x % L;
  const unsigned row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const unsigned n = row % a.N, rest = row / a.N, h = rest % c.H, kv = rest / c.H & 1, z = rest / c.H / 2;
  if (z >= (unsigned)c.Z) return;
  const long long pos = (a.start ? (long long)a.start[z] : 0) + n;
  float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (pos >= 0 && pos < length_of(c, z)) {
    const size_t at = ((size_t)z * c.H + h) * c.C + pos;
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(c.codes[kv]) + at * (D / 8) + lane), p = __ldg(c.param[kv] + at);
    const float s = param_scale(p), zero = param_zero(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = s * ((float)(w >> (4 * i) & 15) - zero);  // 13 bits: exact in fp32
  }
  store8((T*)a.out[kv] + (((size_t)z * c.H + h) * a.N + n) * D + lane * 8, true, y);
}

// ---------------------------------------------------------------- evict
struct EvictArgs {
  Cache from, to;
  int budget, recent;
  int32_t* kept;  // [Z, H, budget]
};

// fp32 as a whole number of the same order; NaN is the largest, -0 is 0
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return ~0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Which positions stay, one CTA per (sequence, head): a radix selection finds
// the least weight that stays (4 passes of 8 bits), then one pass in order
// lists the heavier positions, the first of the equal ones and the last tokens.
constexpr int kSelect = 1024;

__global__ void __launch_bounds__(kSelect) evict_select_kernel(EvictArgs a) {
  __shared__ unsigned hist[256];
  __shared__ unsigned warp_sum[2][32];
  __shared__ unsigned s_prefix, s_left;
  const int zh = blockIdx.x, z = zh / a.from.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = length_of(a.from, z);
  int32_t* kept = a.kept + (size_t)zh * a.budget;
  const float* weight = a.from.weight + (size_t)zh * a.from.C;
  if (zh % a.from.H == 0 && tid == 0) a.to.lens[z] = min(n, a.budget);
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kSelect) kept[i] = i < n ? i : -1;
    return;
  }
  const int old = n - a.recent, need = a.budget - a.recent;
  for (int i = tid; i < a.recent; i += kSelect) kept[need + i] = old + i;
  if (need == 0) return;
  uint32_t prefix = 0, left = need;  // among weights that begin with prefix, the left-th largest is looked for
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < old; i += kSelect) {
      const uint32_t u = order_of(weight[i]);
      if (shift == 24 || u >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[u >> shift & 255], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // lane holds digits 255 - 8 lane .. 248 - 8 lane
      unsigned mine = 0;
      for (int i = 0; i < 8; ++i) mine += hist[255 - 8 * lane - i];
      unsigned sum = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += up;
      }
      unsigned above = sum - mine;
      if (above < left && left <= sum) {
        int d = 255 - 8 * lane;
        while (above + hist[d] < left) above += hist[d--];
        s_prefix = prefix | (uint32_t)d << shift;
        s_left = left - above;
      }
    }
    __syncthreads();
    prefix = s_prefix, left = s_left;
    __syncthreads();
  }
  // `left` of the weights equal to prefix stay: the first ones
  unsigned done = 0, equal = 0;
  for (int i0 = 0; i0 < old; i0 += kSelect) {
    const int i = i0 + tid;
    const uint32_t u = i < old ? order_of(weight[i]) : 0u;
    const bool more = i < old && u > prefix, same = i < old && u == prefix;
    const unsigned bm = __ballot_sync(~0u, more), bs = __ballot_sync(~0u, same), below = (1u << lane) - 1;
    if (lane == 0) warp_sum[0][warp] = __popc(bm), warp_sum[1][warp] = __popc(bs);
    __syncthreads();
    unsigned pm = 0, ps = 0, tm = 0, ts = 0;
    for (int w = 0; w < kSelect / 32; ++w) {
      const unsigned x = warp_sum[0][w], y = warp_sum[1][w];
      if (w < warp) pm += x, ps += y;
      tm += x, ts += y;
    }
    const unsigned em = done + pm + __popc(bm & below), es = equal + ps + __popc(bs & below);
    // rank among the kept: heavier ones before, and equal ones before as far as they stay
    if (more || (same && es < left)) kept[em + min(es, left)] = i;
    done += tm, equal += ts;
    __syncthreads();
  }
}

// Moves what stays: D / 32 lanes of 16 bytes for the key and as many for the value.
template <int D>
__global__ void __launch_bounds__(kThreads) evict_move_kernel(EvictArgs a) {
  constexpr int L = D / 16;
  const Cache &f = a.from, &t = a.to;
  const int zh = blockIdx.y, i = blockIdx.x * (kThreads / L) + threadIdx.x / L, lane = threadIdx.x % L;
  if (i >= a.budget) return;
  const int src = a.kept[(size_t)zh * a.budget + i];
  if (src < 0) return;
  const int kv = lane / (L / 2), part = lane % (L / 2);
  const size_t from = (size_t)zh * f.C + src, to = (size_t)zh * t.C + i;
  reinterpret_cast<uint4*>(t.codes[kv])[to * (D / 32) + part] = __ldg(reinterpret_cast<const uint4*>(f.codes[kv]) + from * (D / 32) + part);
  if (part == 0) {
    t.param[kv][to] = __ldg(f.param[kv] + from);
    if (kv == 0) t.weight[to] = __ldg(f.weight + from);
  }
}

// ------------------------------------------------------------------ host
int check_cache(const qflash_kv4_cache* c, const char* what) {
  if (!c) return set_err(QFLASH_ERR_ARG, "%s: null cache", what);
  if (c->D != 64 && c->D != 128) return set_err(QFLASH_ERR_ARG, "%s: head dim %d not in {64,128}", what, c->D);
  if (c->Z < 0 || c->H < 1 || c->capacity < 1) return set_err(QFLASH_ERR_ARG, "%s: cache of shape %d x %d x %d", what, c->Z, c->H, c->capacity);
  if (c->capacity > 1 << 24) return set_err(QFLASH_ERR_ARG, "%s: capacity %d above 2^24", what, c->capacity);
  if ((long long)c->Z * c->H > 1 << 20) return set_err(QFLASH_ERR_ARG, "%s: %d x %d heads, above 2^20", what, c->Z, c->H);
  if (c->Z == 0) return QFLASH_OK;
  if (!c->k_codes || !c->v_codes || !c->k_param || !c->v_param || !c->weight || !c->lens || !c->ctl)
    return set_err(QFLASH_ERR_ARG, "%s: null pointer in the cache", what);
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15)
    return set_err(QFLASH_ERR_ALIGN, "%s: codes must be 16-byte aligned", what);
  if (((uintptr_t)c->k_param | (uintptr_t)c->v_param | (uintptr_t)c->weight | (uintptr_t)c->lens | (uintptr_t)c->ctl) & 3)
    return set_err(QFLASH_ERR_ALIGN, "%s: parameters, weights and lengths must be 4-byte aligned", what);
  return QFLASH_OK;
}

static size_t elt(int dtype) { return dtype == kF32 ? 4 : 2; }

// rows of 8-element runs can be loaded 16 bytes at a time
static bool aligned16(const void* p, const int64_t st[4], int dtype) {
  const size_t e = elt(dtype);
  return (((uintptr_t)p | (st[0] * e) | (st[1] * e) | (st[2] * e)) & 15) == 0;
}

static bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

template <class T>
static int launch_append(const AppendArgs& a, cudaStream_t s) {
  const unsigned per = kThreads / (a.c.D / 8);
  const unsigned grid = (unsigned)((2LL * a.c.Z * a.c.H * a.N + per - 1) / per);
  if (a.c.D == 64)
    append_kernel<T, 64><<<grid, kThreads, 0, s>>>(a);
  else
    append_kernel<T, 128><<<grid, kThreads, 0, s>>>(a);
  return check_launch("kv4 append", grid);
}

template <class T>
static int launch_read(const ReadArgs& a, cudaStream_t s) {
  const unsigned per = kThreads / (a.c.D / 8);
  const unsigned grid = (unsigned)((2LL * a.c.Z * a.c.H * a.N + per - 1) / per);
  if (a.c.D == 64)
    read_kernel<T, 64><<<grid, kThreads, 0, s>>>(a);
  else
    read_kernel<T, 128><<<grid, kThreads, 0, s>>>(a);
  return check_launch("kv4 read", grid);
}

}  // namespace kv4
}  // namespace qfb

using namespace qfb;
using namespace qfb::kv4;

extern "C" int qflash_kv4_append(const qflash_kv4_cache* cache, const void* k, const void* v, int dtype,
                                 const int64_t k_strides[4], const int64_t v_strides[4], int N,
                                 const int32_t* new_lens, const int32_t* at, void* stream) {
  if (int rc = check_cache(cache, "kv4 append")) return rc;
  if (N < 0) return set_err(QFLASH_ERR_ARG, "kv4 append: negative N");
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return set_err(QFLASH_ERR_ARG, "kv4 append: dtype %d", dtype);
  if (2LL * cache->Z * cache->H * N >= 1LL << 31) return set_err(QFLASH_ERR_UNSUPPORTED, "kv4 append: 2^31 vectors or more");
  if (cache->Z == 0 || N == 0) return QFLASH_OK;
  if (!k || !v || !k_strides || !v_strides) return set_err(QFLASH_ERR_ARG, "kv4 append: null pointer");
  if (k_strides[3] != 1 || v_strides[3] != 1) return set_err(QFLASH_ERR_ARG, "kv4 append: innermost (head-dim) stride must be 1");
  DeviceGuard keep_device;
  int dev = 0;
  if (int rc = select_device(cache->k_codes, &dev)) return rc;
  AppendArgs a;
  a.c = view(cache);
  a.x[0] = k, a.x[1] = v;
  for (int i = 0; i < 3; ++i) a.st[0][i] = k_strides[i], a.st[1][i] = v_strides[i];
  a.vec[0] = aligned16(k, k_strides, dtype), a.vec[1] = aligned16(v, v_strides, dtype);
  a.N = N, a.new_lens = new_lens, a.at = at;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == kF32 ? launch_append<float>(a, s) : dtype == kF16 ? launch_append<__half>(a, s) : launch_append<__nv_bfloat16>(a, s);
}

extern "C" int qflash_kv4_read(const qflash_kv4_cache* cache, void* k, void* v, int dtype, int N, const int32_t* start,
                               void* stream) {
  if (int rc = check_cache(cache, "kv4 read")) return rc;
  if (N < 0) return set_err(QFLASH_ERR_ARG, "kv4 read: negative N");
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return set_err(QFLASH_ERR_ARG, "kv4 read: dtype %d", dtype);
  if (2LL * cache->Z * cache->H * N >= 1LL << 31) return set_err(QFLASH_ERR_UNSUPPORTED, "kv4 read: 2^31 vectors or more");
  if (cache->Z == 0 || N == 0) return QFLASH_OK;
  if (!k || !v) return set_err(QFLASH_ERR_ARG, "kv4 read: null pointer");
  if (((uintptr_t)k | (uintptr_t)v) & 15) return set_err(QFLASH_ERR_ALIGN, "kv4 read: outputs must be 16-byte aligned");
  DeviceGuard keep_device;
  int dev = 0;
  if (int rc = select_device(cache->k_codes, &dev)) return rc;
  const ReadArgs a = {view(cache), {k, v}, N, start};
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == kF32 ? launch_read<float>(a, s) : dtype == kF16 ? launch_read<__half>(a, s) : launch_read<__nv_bfloat16>(a, s);
}

extern "C" int qflash_kv4_evict(const qflash_kv4_cache* from, const qflash_kv4_cache* to, int budget, int recent,
                                int32_t* kept, void* stream) {
  if (int rc = check_cache(from, "kv4 evict")) return rc;
  if (int rc = check_cache(to, "kv4 evict")) return rc;
  if (from->Z != to->Z || from->H != to->H || from->D != to->D)
    return set_err(QFLASH_ERR_ARG, "kv4 evict: caches of %d x %d heads of %d and of %d x %d heads of %d", from->Z, from->H,
                   from->D, to->Z, to->H, to->D);
  if (budget < 1 || budget > to->capacity) return set_err(QFLASH_ERR_ARG, "kv4 evict: budget %d of a capacity of %d", budget, to->capacity);
  if (recent < 0 || recent > budget) return set_err(QFLASH_ERR_ARG, "kv4 evict: %d recent tokens of a budget of %d", recent, budget);
  if (from->Z == 0) return QFLASH_OK;
  if (!kept) return set_err(QFLASH_ERR_ARG, "kv4 evict: null pointer");
  const size_t heads = (size_t)from->Z * from->H, fc = heads * from->capacity, tc = heads * to->capacity;
  const struct { const void *a, *b; size_t bytes; } bufs[] = {
      {from->k_codes, to->k_codes, (size_t)from->D / 2}, {from->v_codes, to->v_codes, (size_t)from->D / 2},
      {from->k_param, to->k_param, 4}, {from->v_param, to->v_param, 4}, {from->weight, to->weight, 4}};
  for (const auto& x : bufs)
    for (const auto& y : bufs)
      if (overlap(x.a, fc * x.bytes, y.b, tc * y.bytes))
        return set_err(QFLASH_ERR_ARG, "kv4 evict: the caches share memory");
  if (overlap(from->lens, 4 * (size_t)from->Z, to->lens, 4 * (size_t)to->Z)) return set_err(QFLASH_ERR_ARG, "kv4 evict: the caches share memory");
  DeviceGuard keep_device;
  int dev = 0;
  if (int rc = select_device(from->k_codes, &dev)) return rc;
  const EvictArgs a = {view(from), view(to), budget, recent, kept};
  cudaStream_t s = (cudaStream_t)stream;
  evict_select_kernel<<<(unsigned)heads, kSelect, 0, s>>>(a);
  if (int rc = check_launch("kv4 evict select", (unsigned)heads)) return rc;
  const int per = kThreads / (from->D / 16);
  const unsigned nx = (unsigned)((budget + per - 1) / per);
  for (size_t h0 = 0; h0 < heads; h0 += 65535) {
    EvictArgs b = a;
    const size_t n = std::min<size_t>(65535, heads - h0);
    for (int i = 0; i < 2; ++i) {
      b.from.codes[i] += h0 * from->capacity * (from->D / 2), b.to.codes[i] += h0 * to->capacity * (to->D / 2);
      b.from.param[i] += h0 * from->capacity, b.to.param[i] += h0 * to->capacity;
    }
    b.from.weight += h0 * from->capacity, b.to.weight += h0 * to->capacity, b.kept += h0 * budget;
    if (from->D == 64)
      evict_move_kernel<64><<<dim3(nx, (unsigned)n), kThreads, 0, s>>>(b);
    else
      evict_move_kernel<128><<<dim3(nx, (unsigned)n), kThreads, 0, s>>>(b);
    if (int rc = check_launch("kv4 evict move", nx)) return rc;
  }
  return QFLASH_OK;
}

static int check_attend(const qflash_kv4_cache* cache, int dtype, int Hq, int N) {
  if (int rc = check_cache(cache, "kv4 attend")) return rc;
  if (dtype != kF16 && dtype != kBF16) return set_err(QFLASH_ERR_ARG, "kv4 attend: queries are fp16 or bf16 (dtype %d)", dtype);
  if (N < 0) return set_err(QFLASH_ERR_ARG, "kv4 attend: negative N");
  if (Hq < 1 || Hq % cache->H) return set_err(QFLASH_ERR_ARG, "kv4 attend: %d query heads over %d key/value heads", Hq, cache->H);
  if (Hq / cache->H > 64) return set_err(QFLASH_ERR_UNSUPPORTED, "kv4 attend: %d query heads per key/value head, above 64", Hq / cache->H);
  if ((long long)Hq / cache->H * N >= 1LL << 24) return set_err(QFLASH_ERR_UNSUPPORTED, "kv4 attend: 2^24 rows per head or more");
  return QFLASH_OK;
}

// Rows of a head from which the kernel for many rows is used.
static bool many_rows(const qflash_kv4_cache* c, int Hq, int N) { return (long long)Hq / c->H * N > 64; }

static size_t attend_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  return many_rows(c, Hq, N) ? prompt_workspace(c, Hq, N, weights) : rows_workspace(c, Hq, N, weights);
}

extern "C" size_t qflash_kv4_attend_workspace(const qflash_kv4_cache* cache, int dtype, int Hq, int N, int weights) {
  if (check_attend(cache, dtype, Hq, N) || cache->Z == 0 || N == 0) return 0;
  return attend_workspace(cache, Hq, N, weights != 0);
}

extern "C" int qflash_kv4_attend(const qflash_kv4_cache* cache, const void* q, int dtype, const int64_t q_strides[4],
                                 void* out, const int64_t out_strides[4], int Hq, int N, const int32_t* new_lens,
                                 double scale, int causal, const float* weights_in, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (int rc = check_attend(cache, dtype, Hq, N)) return rc;
  if (!std::isfinite(scale)) return set_err(QFLASH_ERR_ARG, "kv4 attend: scale is not finite");
  if (cache->Z == 0 || N == 0) return QFLASH_OK;
  if (!q || !out || !q_strides || !out_strides) return set_err(QFLASH_ERR_ARG, "kv4 attend: null pointer");
  if (q_strides[3] != 1 || out_strides[3] != 1) return set_err(QFLASH_ERR_ARG, "kv4 attend: innermost (head-dim) stride must be 1");
  const size_t need = attend_workspace(cache, Hq, N, weights_in != nullptr);
  if (!workspace || workspace_bytes < need)
    return set_err(QFLASH_ERR_ARG, "kv4 attend: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return set_err(QFLASH_ERR_ALIGN, "kv4 attend: workspace must be 16-byte aligned");
  DeviceGuard keep_device;
  int dev = 0;
  if (int rc = select_device(cache->k_codes, &dev)) return rc;
  AttendArgs a;
  a.c = view(cache);
  a.q = q, a.out = out;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.os[i] = out_strides[i];
  a.rep = Hq / cache->H, a.N = N, a.new_lens = new_lens, a.causal = causal;
  a.scale_log2e = (float)(scale * 1.4426950408889634);
  a.weights_in = weights_in;
  a.tok0 = 0, a.ntok = N;
  return many_rows(cache, Hq, N) ? attend_prompt(a, dtype == kF16, workspace, dev, (cudaStream_t)stream)
                                 : attend_rows(a, dtype == kF16, workspace, dev, (cudaStream_t)stream);
}
