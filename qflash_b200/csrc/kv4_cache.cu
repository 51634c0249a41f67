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
#include <atomic>
#include <type_traits>

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
constexpr int kThreads = 256;

// How threads are shared out: a unit is the keys or the values of a (sequence,
// head), unit = (z H + h) 2 + kv, and is worked on by 2^log_group threads of a
// block, so that neither a single token nor a prompt leaves threads idle and no
// thread divides but once.
struct Share {
  int log_group, units;
  // One resident wave of blocks, which go on to further parts of their units: a block's beginning and end
  // (lengths, the ticket) cost several microseconds of latency.  work: threads' worth of a unit.
  dim3 grid(long long work, int per_thread, int blocks) const {
    const long long group = 1LL << log_group;
    const unsigned x = (unsigned)((units + (kThreads >> log_group) - 1) / (kThreads >> log_group));
    const long long parts = (work + group * per_thread - 1) / (group * per_thread);
    return dim3(x, (unsigned)std::max(1LL, std::min<long long>(std::min<long long>(parts, 65535), blocks / x)));
  }
};
static Share share(long long work, long long units, int least) {
  int lg = 0;
  while ((1 << lg) < kThreads && (1LL << lg) < std::max<long long>(work, least)) ++lg;
  return {lg, (int)units};
}

struct AppendArgs {
  Cache c;
  const void* x[2];
  int64_t st[2][3];
  int N;
  const int32_t* new_lens;
  const int32_t* at;
  bool vec[2];
  Share share;
};

// bf16(fp32((hi - lo) / 15)).  The fp32 product is off by at most 3 units in the
// last place, so only one that lies near a border between bf16 numbers has to be
// formed in fp64.
__device__ __forceinline__ float scale_of(float lo, float hi) {
  const float q = (hi - lo) * (1.f / 15.f);
  const int below = (int)(__float_as_uint(q) & 0xffffu) - 0x8000;
  if (q > 1e-30f && q < 1e30f && (below > 8 || below < -8)) return __bfloat162float(__float2bfloat16_rn(q));
  return __bfloat162float(__float2bfloat16_rn((float)(((double)hi - (double)lo) / 15.0)));
}

// rint(fp32(x / s)) for x and s of 16 bits, and their quotient below 32: t = x inv is
// off by a few 2^-23 of itself, and the residual x - t s, exact in one fma, takes that
// to 2^-44.  A quotient n + 1/2 is then hit exactly, and any other quotient of
// numbers of 11 and 8 bits lies further than that from n + 1/2 (by 2^-17 of itself
// at least), so rounding it is rounding the exact quotient, and so is rounding the fp32 one.
__device__ __forceinline__ float quotient16(float x, float s, float inv) {
  const float t = x * inv;
  return __fmaf_rn(__fmaf_rn(-t, s, x), inv, t);
}
constexpr float kRound = 12582912.f;  // 1.5 2^23: adding it rounds to even like rint, the whole number in the low bits

// The codes of 8 quotients, clamp(rint(q) + zero, 0, 15), one to 4 bits.
__device__ __forceinline__ uint32_t codes_of(const float (&q)[8], float zero) {
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)  // clamp first, between whole numbers; then sums mod 2^32 of what lies above the rounding constant
    word += __float_as_uint(__fadd_rn(fminf(fmaxf(q[i], -zero), 15.f - zero), kRound)) << (4 * i);
  return word + ((uint32_t)(int)zero - 0x4b400000u) * 0x11111111u;  // 0x4b400000: kRound's bits
}

// Least and greatest of 8 elements and 0.  16-bit elements in pairs; NaN stays.
template <class T>
__device__ __forceinline__ void range8(const T (&r)[8], float& lo, float& hi) {
  if constexpr (sizeof(T) == 4) {
    lo = hi = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(r[i]));
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(r[i]));
    }
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
    uint32_t l = 0, h = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(l) : "r"(w[i]));
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(h) : "r"(w[i]));
      } else {
        asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(l) : "r"(w[i]));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(h) : "r"(w[i]));
      }
    }
    const T* lp = reinterpret_cast<const T*>(&l);
    const T* hp = reinterpret_cast<const T*>(&h);
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(lo) : "f"(to_float(lp[0])), "f"(to_float(lp[1])));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(hi) : "f"(to_float(hp[0])), "f"(to_float(hp[1])));
  }
}

// D / 8 lanes per vector, 8 elements each; a thread holds U vectors' elements at
// once, so that loads are under way while others are worked on.  Two prompts of up to
// 8191 tokens, 8 heads of 128, fp16 (67 MB in, 18 MB out): 33 us, 2.5 TB/s; instructions
// bound it (70 % of issue slots): 9 quotients per 8 elements, each with a residual, where
// fp32 divisions took 56 us.  One token of 32 sequences: 3.7 us, of which launch and ticket are most.
template <class T, int D, int U>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a) {
  constexpr int L = D / 8;
  const Cache& c = a.c;
  const int lg = a.share.log_group, in_group = threadIdx.x & ((1 << lg) - 1), lane = threadIdx.x % L;
  const int unit = blockIdx.x * (kThreads >> lg) + (threadIdx.x >> lg);
  const bool there = unit < a.share.units;
  const int kv = unit & 1, zh = min(unit, a.share.units - 1) >> 1, z = zh / c.H, h = zh - z * c.H;
  const int base = a.at ? a.at[z] : length_of(c, z);
  const int fresh = there ? (a.new_lens ? min(max(a.new_lens[z], 0), a.N) : a.N) : 0;
  const T* x0 = (const T*)(kv ? a.x[1] : a.x[0]) + z * (kv ? a.st[1][0] : a.st[0][0]) + h * (kv ? a.st[1][1] : a.st[0][1]) + lane * 8;
  const int64_t x_step = kv ? a.st[1][2] : a.st[0][2];
  const bool vec = kv ? a.vec[1] : a.vec[0];
  uint32_t* codes = reinterpret_cast<uint32_t*>(kv ? c.codes[1] : c.codes[0]);
  uint32_t* param = kv ? c.param[1] : c.param[0];
  const size_t head = (size_t)zh * c.C;
  const int per = (1 << lg) / L;  // vectors of a group's step
  const unsigned group = (L == 32 ? ~0u : (1u << L) - 1) << (threadIdx.x % 32 / L * L);
  for (int n0 = (blockIdx.y * U) * per + in_group / L; n0 < fresh; n0 += gridDim.y * U * per) {
    alignas(16) T r[U][8];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + u * per;
      const long long pos = (long long)base + n;
      in[u] = n < fresh && pos >= 0 && pos < c.C;
      if (in[u]) {
        const T* from = x0 + n * x_step;
        if (vec) {
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4*>(r[u])[i] = __ldg(reinterpret_cast<const uint4*>(from) + i);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) r[u][i] = from[i];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in[u]) continue;  // the vector's lanes together
      float lo, hi;
      range8(r[u], lo, hi);
#pragma unroll
      for (int o = L / 2; o; o >>= 1) {
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(__shfl_xor_sync(group, lo, o)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(__shfl_xor_sync(group, hi, o)));
      }
      const bool good = lo > -INFINITY && hi < INFINITY;  // no infinity, no NaN
      const float s = good ? scale_of(lo, hi) : __uint_as_float(0x7fc00000u);
      float zero = 0.f;
      uint32_t word = 0;
      if (s > 0.f) {
        float inv, q[8];
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        if (sizeof(T) == 2 && s > 1e-30f && s < 1e30f) {
          zero = quotient16(-lo, s, inv);
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = quotient16(to_float(r[u][i]), s, inv);
        } else {  // fp32 elements: only a product near to a border needs the division itself
          zero = __fdiv_rn(-lo, s);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = to_float(r[u][i]);
            q[i] = x * inv;
            if (!(s > 1e-30f && s < 1e30f && fabsf(q[i] - rintf(q[i])) < 0.5f - 1e-5f)) q[i] = __fdiv_rn(x, s);
          }
        }
        zero = fminf(fmaxf(rintf(zero), 0.f), 15.f);
        word = codes_of(q, zero);
      }
      const size_t to = head + (base + n0 + u * per);
      codes[to * L + lane] = word;
      if (lane == 0) {
        param[to] = __float_as_uint(s) >> 16 | __float_as_uint(zero) & 0xffff0000u;
        if (kv == 0) c.weight[to] = 0.f;
      }
    }
  }
  // The last CTA moves lens on, after every CTA has read them.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&c.ctl[0], 1) == (int)(gridDim.x * gridDim.y) - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int i = threadIdx.x; i < c.Z; i += kThreads) {
    const int first = a.at ? a.at[i] : length_of(c, i);
    const long long end = (long long)first + (a.new_lens ? min(max(a.new_lens[i], 0), a.N) : a.N);
    if (first < 0 || end > c.C) atomicOr(&c.ctl[1], 1);
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
  Share share;
};

__device__ __forceinline__ uint32_t pair_sub(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("sub.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ uint32_t pair_mul(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// The 8 values of a word of codes.  code - zero is exact in bf16 (set into the
// mantissa of 128), and so is scale * (code - zero) in fp32: one rounding, to T.
template <class T>
__device__ __forceinline__ void put_values(T* out, uint32_t w, uint32_t param) {
  const uint32_t z1 = __float_as_uint(128.f + param_zero(param)) >> 16, zero = z1 | z1 << 16;
  uint32_t y[4];  // elements i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = pair_sub(w >> (4 * i) & 0x000f000fu | 0x43004300u, zero);
  if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
    const uint32_t s = __byte_perm(param, param, 0x1010);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = pair_mul(y[i], s);
    *reinterpret_cast<uint4*>(out) = make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410),
                                                __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632));
  } else {
    const float s = param_scale(param);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = s * __uint_as_float(y[i] << 16);
      x[i + 4] = s * __uint_as_float(y[i] & 0xffff0000u);
    }
    store8(out, true, x);
  }
}

// A unit's words are in one run, and so are its values: a thread takes U words
// of 8 codes (coalesced 4 bytes in, 16 out), loads before stores.  4 sequences of up to
// 8192 positions, 8 heads of 64, bf16: 16.4 us, 4.6 TB/s, three quarters of it writes, which bound it.
template <class T, int D, int U>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs a) {
  constexpr int L = D / 8;
  const Cache& c = a.c;
  const int lg = a.share.log_group, in_group = threadIdx.x & ((1 << lg) - 1);
  const int unit = blockIdx.x * (kThreads >> lg) + (threadIdx.x >> lg);
  if (unit >= a.share.units) return;
  const int kv = unit & 1, zh = unit >> 1, z = zh / c.H;
  const int first = a.start ? a.start[z] : 0, len = length_of(c, z);
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(kv ? c.codes[1] : c.codes[0]) + (size_t)zh * c.C * L;
  const uint32_t* param = (kv ? c.param[1] : c.param[0]) + (size_t)zh * c.C;
  T* out = (T*)(kv ? a.out[1] : a.out[0]) + (size_t)zh * a.N * D;
  const long long words = (long long)a.N * L, step = (long long)gridDim.y * U << lg;
  for (long long w0 = ((long long)blockIdx.y * U << lg) + in_group; w0 < words; w0 += step) {
    uint32_t w[U], p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = w0 + ((long long)u << lg), pos = first + i / L;
      const bool in = i < words && pos >= 0 && pos < len;
      w[u] = in ? __ldg(codes + pos * L + i % L) : 0u;
      p[u] = in ? __ldg(param + pos) : 0u;  // scale 0
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = w0 + ((long long)u << lg);
      if (i < words) put_values(out + i * 8, w[u], p[u]);
    }
  }
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

// Which positions stay, a cluster of CTAs per (sequence, head), each with a run
// of the positions: a radix selection over digits of 11, 11 and 10 bits finds the
// least weight that stays, then the heavier positions, the first of the equal ones
// and the last tokens are listed in order.  The CTAs add up their counts through
// shared memory of the cluster.  A run of up to 16384 positions is read once and
// kept in registers; latency bounds this kernel, not bytes: three digits with a cluster
// barrier or more each.  8 heads of 131071 positions 20 us (one CTA a head that reads them for each digit 348),
// 128 heads of up to 4300 10.6 us.
constexpr int kSelect = 1024;
constexpr int kKeep = 16;  // positions per thread and tile
constexpr int kDigits = 2048;
constexpr int kCluster = 8;

// A word of CTA `rank` of the cluster, or of this one if it is alone.
__device__ __forceinline__ uint32_t word_of(const uint32_t* p, int rank, int cs) { return cs > 1 ? peer_word(p, rank) : *p; }

// The sum of a word over the cluster, all loads under way before the first is added.
__device__ __forceinline__ uint32_t cluster_sum(const uint32_t* p, int cs) {
  uint32_t x[kCluster], sum = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) x[r] = r < cs ? word_of(p, r, cs) : 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) sum += x[r];
  return sum;
}

__device__ __forceinline__ uint32_t warp_scan(uint32_t x) {  // of this lane and those below
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(~0u, x, o);
    if ((threadIdx.x & 31) >= o) x += up;
  }
  return x;
}

__global__ void __launch_bounds__(kSelect) evict_select_kernel(EvictArgs a) {
  constexpr int W = kSelect / 32, GROUPS = kDigits / 32;
  __shared__ uint32_t hist[2][kDigits];  // of even and odd passes: peers may still read the last pass's
  __shared__ uint32_t coarse[2][GROUPS];  // sums of 32 digits
  __shared__ uint32_t counts[2], s_digit, s_left;
  __shared__ uint32_t warp_more[W], warp_same[W];
  may_begin();
  const int cs = (int)cluster_size(), rank = (int)cluster_rank();
  const int zh = blockIdx.x / cs, z = zh / a.from.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = length_of(a.from, z);
  int32_t* kept = a.kept + (size_t)zh * a.budget;
  const float* weight = a.from.weight + (size_t)zh * a.from.C;
  if (zh % a.from.H == 0 && rank == 0 && tid == 0) a.to.lens[z] = min(n, a.budget);
  const int stride = cs * kSelect, mine = rank * kSelect + tid;
  if (n <= a.budget) {  // all CTAs of the cluster return together
    for (int i = mine; i < a.budget; i += stride) kept[i] = i < n ? i : -1;
    return;
  }
  const int old = n - a.recent, need = a.budget - a.recent;
  for (int i = mine; i < a.recent; i += stride) kept[need + i] = old + i;
  if (need == 0) return;
  const int run = (old + cs - 1) / cs, i0 = min(old, rank * run), i1 = min(old, i0 + run);
  // a thread holds `keep` positions of a tile in u, a warp's are neighbours: at(t, j), j < keep
  const int keep = min(kKeep, (run + kSelect - 1) / kSelect), tile = kSelect * keep;
  const bool once = run <= tile;
  uint32_t u[kKeep];
  auto at = [&](int t, int j) { return i0 + t * tile + (warp * keep + j) * 32 + lane; };
  auto load = [&](int t) {
    float w[kKeep];
#pragma unroll
    for (int j = 0; j < kKeep; ++j) w[j] = j < keep && at(t, j) < i1 ? __ldg(weight + at(t, j)) : 0.f;
#pragma unroll
    for (int j = 0; j < kKeep; ++j) u[j] = order_of(w[j]);
  };
  const int tiles = (i1 - i0 + tile - 1) / tile;
  uint32_t prefix = 0, left = need;  // among weights that begin with prefix, the left-th largest is looked for
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    uint32_t *h = hist[pass & 1], *hc = coarse[pass & 1];
    for (int i = tid; i < kDigits; i += kSelect) h[i] = 0;
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
      if (pass == 0 || !once) load(t);
#pragma unroll
      for (int j = 0; j < kKeep; ++j) {
        if (j >= keep) break;
        if (at(t, j) < i1 && (pass == 0 || u[j] >> (shift + bits) == prefix >> (shift + bits)))
          atomicAdd(&h[u[j] >> shift & ((1 << bits) - 1)], 1u);
      }
    }
    __syncthreads();
    for (int i = warp; i < GROUPS; i += W) {
      const uint32_t sum = __reduce_add_sync(~0u, h[32 * i + lane]);
      if (lane == 0) hc[i] = sum;
    }
    if (cs > 1) cluster_sync(); else __syncthreads();
    if (warp == 0) {
      // from the top: the group of 32 digits, two to a lane, then the digit, so that little crosses the cluster
      const uint32_t g0 = cluster_sum(hc + GROUPS - 1 - 2 * lane, cs), g1 = cluster_sum(hc + GROUPS - 2 - 2 * lane, cs);
      const uint32_t upto = warp_scan(g0 + g1), before = upto - g0 - g1;
      const bool first = before < left && left <= before + g0, second = before + g0 < left && left <= upto;
      const int l = __ffs(__ballot_sync(~0u, first || second)) - 1;
      const int group = __shfl_sync(~0u, GROUPS - 1 - 2 * lane - (second ? 1 : 0), l);
      const uint32_t above = __shfl_sync(~0u, before + (second ? g0 : 0), l);
      const int digit = 32 * group + 31 - lane;
      const uint32_t d = cluster_sum(h + digit, cs), to = above + warp_scan(d);
      if (to - d < left && left <= to) s_digit = digit, s_left = left - (to - d);
    }
    __syncthreads();
    prefix |= s_digit << shift, left = s_left;
  }
  // heavier and equal positions of a warp's part of a tile
  auto count = [&](int t, uint32_t& more, uint32_t& same) {
    uint32_t m = 0, e = 0;
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
      if (j >= keep) break;
      m += at(t, j) < i1 && u[j] > prefix;
      e += at(t, j) < i1 && u[j] == prefix;
    }
    more = __reduce_add_sync(~0u, m), same = __reduce_add_sync(~0u, e);
  };
  // how many of them the CTAs before this one have
  uint32_t done = 0, equal = 0, more = 0, same = 0;
  if (cs > 1) {
    for (int t = 0; t < tiles; ++t) {
      if (!once) load(t);
      count(t, more, same);
      if (lane == 0) atomicAdd(&counts[0], more), atomicAdd(&counts[1], same);
    }
    cluster_sync();
    uint32_t x[2] = {0, 0};
    if (lane < 2 * rank) x[lane & 1] = peer_word(&counts[lane & 1], lane >> 1);
    done = __reduce_add_sync(~0u, x[0]), equal = __reduce_add_sync(~0u, x[1]);
  }
  for (int t = 0; t < tiles; ++t) {
    if (!once) load(t);
    if (cs == 1 || !once) count(t, more, same);
    if (lane == 0) warp_more[warp] = more, warp_same[warp] = same;
    __syncthreads();
    const uint32_t m = warp_more[lane], e = warp_same[lane];  // kSelect / 32 is 32
    uint32_t pm = done + __reduce_add_sync(~0u, lane < warp ? m : 0u), ps = equal + __reduce_add_sync(~0u, lane < warp ? e : 0u);
    done += __reduce_add_sync(~0u, m), equal += __reduce_add_sync(~0u, e);
    const unsigned below = (1u << lane) - 1;
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
      if (j >= keep) break;
      const bool in = at(t, j) < i1, heavy = in && u[j] > prefix, even = in && u[j] == prefix;
      const unsigned bm = __ballot_sync(~0u, heavy), be = __ballot_sync(~0u, even);
      const uint32_t em = pm + __popc(bm & below), es = ps + __popc(be & below);
      // rank among the kept: heavier ones before, and equal ones before as far as they stay
      // (never past `need`, unless the weights change meanwhile)
      if ((heavy || (even && es < left)) && em + min(es, left) < (uint32_t)need) kept[em + min(es, left)] = at(t, j);
      pm += __popc(bm), ps += __popc(be);
    }
    __syncthreads();
  }
  if (cs > 1) cluster_sync();  // no CTA's shared memory goes while a peer may read it
}

// Moves what stays: D / 32 lanes of 16 bytes for the key and as many for the
// value, kMove positions at once, since a position's address comes from a load.  128 heads
// keeping up to 2048 of 4300 positions of 128: about 15 us for 71 MB at most; 8 heads keeping 8192: 7 us.
constexpr int kMove = 4;
template <int D>
__global__ void __launch_bounds__(kThreads) evict_move_kernel(EvictArgs a) {
  constexpr int L = D / 16, G = kThreads / L;
  const Cache &f = a.from, &t = a.to;
  const int zh = blockIdx.y, i0 = blockIdx.x * (G * kMove) + threadIdx.x / L, lane = threadIdx.x % L;
  const int kv = lane / (L / 2), part = lane % (L / 2);
  const uint4* from = reinterpret_cast<const uint4*>(kv ? f.codes[1] : f.codes[0]) + (size_t)zh * f.C * (D / 32) + part;
  uint4* to = reinterpret_cast<uint4*>(kv ? t.codes[1] : t.codes[0]) + (size_t)zh * t.C * (D / 32) + part;
  const uint32_t* from_param = (kv ? f.param[1] : f.param[0]) + (size_t)zh * f.C;
  uint32_t* to_param = (kv ? t.param[1] : t.param[0]) + (size_t)zh * t.C;
  wait_for_previous();
  int src[kMove];
  uint4 x[kMove];
  uint32_t p[kMove];
  float w[kMove];
#pragma unroll
  for (int k = 0; k < kMove; ++k) src[k] = i0 + k * G < a.budget ? a.kept[(size_t)zh * a.budget + i0 + k * G] : -1;
#pragma unroll
  for (int k = 0; k < kMove; ++k)
    if (src[k] >= f.C) src[k] = -1;  // as kept is where weights changed meanwhile
#pragma unroll
  for (int k = 0; k < kMove; ++k)
    if (src[k] >= 0) {
      x[k] = __ldg(from + (size_t)src[k] * (D / 32));
      if (part == 0) p[k] = __ldg(from_param + src[k]);
      if (lane == 0) w[k] = __ldg(f.weight + (size_t)zh * f.C + src[k]);
    }
#pragma unroll
  for (int k = 0; k < kMove; ++k)
    if (src[k] >= 0) {
      const int i = i0 + k * G;
      to[(size_t)i * (D / 32)] = x[k];
      if (part == 0) to_param[i] = p[k];
      if (lane == 0) t.weight[(size_t)zh * t.C + i] = w[k];
    }
}

// What attend leaves of the weights where it has no rows: those that it was given, for stored positions.
__global__ void __launch_bounds__(kThreads) set_weights_kernel(Cache c, const float* from, int parts) {
  const int zh = blockIdx.x / parts, len = length_of(c, zh / c.H);
  const size_t head = (size_t)zh * c.C;
  for (int j = blockIdx.x % parts * kThreads + threadIdx.x; j < len; j += parts * kThreads) c.weight[head + j] = from[head + j];
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

// Makes the cache's device current for a call's launches, and the caller's again behind them.
struct OnDevice {
  int prev = -1, dev = 0, rc = QFLASH_OK;
  explicit OnDevice(const qflash_kv4_cache* c) {
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess) {
      cudaGetLastError();
      cur = -1;
    }
    if (c->device == cur && cur >= 0 && known(cur)) {
      dev = cur;
      return;
    }
    prev = cur;
    rc = select_device(c->k_codes, &dev);
    if (!rc && c->device >= 0 && c->device != dev)
      rc = set_err(QFLASH_ERR_ARG, "kv4: the cache's buffers are on device %d, not %d", dev, c->device);
    if (!rc) seen()[dev].store(true, std::memory_order_relaxed);
  }
  ~OnDevice() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  static std::atomic<bool>* seen() {  // devices that select_device has accepted
    static std::atomic<bool> s[kDevices];
    return s;
  }
  static bool known(int d) { return d < kDevices && seen()[d].load(std::memory_order_relaxed); }
};

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
static int launch_append(AppendArgs& a, int sms, cudaStream_t s) {
  const int L = a.c.D / 8;
  constexpr int U = 2;
  a.share = share((long long)a.N * L, 2LL * a.c.Z * a.c.H, L);
  const dim3 grid = a.share.grid((long long)a.N * L, U, sms * 5);
  if (a.c.D == 64)
    append_kernel<T, 64, U><<<grid, kThreads, 0, s>>>(a);
  else
    append_kernel<T, 128, U><<<grid, kThreads, 0, s>>>(a);
  return check_launch("kv4 append", grid.x * grid.y);
}

template <class T>
static int launch_read(ReadArgs& a, int sms, cudaStream_t s) {
  const int L = a.c.D / 8;
  constexpr int U = 4;
  a.share = share((long long)a.N * L, 2LL * a.c.Z * a.c.H, L);
  const dim3 grid = a.share.grid((long long)a.N * L, U, sms * 8);
  if (a.c.D == 64)
    read_kernel<T, 64, U><<<grid, kThreads, 0, s>>>(a);
  else
    read_kernel<T, 128, U><<<grid, kThreads, 0, s>>>(a);
  return check_launch("kv4 read", grid.x * grid.y);
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
  if (cache->Z == 0 || (N == 0 && !at)) return QFLASH_OK;
  if ((N && (!k || !v)) || !k_strides || !v_strides) return set_err(QFLASH_ERR_ARG, "kv4 append: null pointer");
  if (N && (k_strides[3] != 1 || v_strides[3] != 1)) return set_err(QFLASH_ERR_ARG, "kv4 append: innermost (head-dim) stride must be 1");
  OnDevice on(cache);
  if (on.rc) return on.rc;
  const int dev = on.dev;
  AppendArgs a;
  a.c = view(cache);
  a.x[0] = k, a.x[1] = v;
  for (int i = 0; i < 3; ++i) a.st[0][i] = k_strides[i], a.st[1][i] = v_strides[i];
  a.vec[0] = aligned16(k, k_strides, dtype), a.vec[1] = aligned16(v, v_strides, dtype);
  a.N = N, a.new_lens = new_lens, a.at = at;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == kF32 ? launch_append<float>(a, sm_count(dev), s) : dtype == kF16 ? launch_append<__half>(a, sm_count(dev), s) : launch_append<__nv_bfloat16>(a, sm_count(dev), s);
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
  OnDevice on(cache);
  if (on.rc) return on.rc;
  const int dev = on.dev;
  ReadArgs a = {view(cache), {k, v}, N, start, {}};
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == kF32 ? launch_read<float>(a, sm_count(dev), s) : dtype == kF16 ? launch_read<__half>(a, sm_count(dev), s) : launch_read<__nv_bfloat16>(a, sm_count(dev), s);
}

extern "C" int qflash_kv4_evict(const qflash_kv4_cache* from, const qflash_kv4_cache* to, int budget, int recent,
                                int32_t* kept, void* stream) {
  if (int rc = check_cache(from, "kv4 evict")) return rc;
  if (int rc = check_cache(to, "kv4 evict")) return rc;
  if (from->Z != to->Z || from->H != to->H || from->D != to->D)
    return set_err(QFLASH_ERR_ARG, "kv4 evict: caches of %d x %d heads of %d and of %d x %d heads of %d", from->Z, from->H,
                   from->D, to->Z, to->H, to->D);
  if (from->device >= 0 && to->device >= 0 && from->device != to->device)
    return set_err(QFLASH_ERR_ARG, "kv4 evict: caches on devices %d and %d", from->device, to->device);
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
  OnDevice on(from);
  if (on.rc) return on.rc;
  const int dev = on.dev;
  if (to->device != dev) {
    int there = -1;
    const int rc = select_device(to->k_codes, &there);  // which makes it the current one
    if (there != dev) cudaSetDevice(dev);
    if (rc) return rc;
    if (there != dev) return set_err(QFLASH_ERR_ARG, "kv4 evict: caches on devices %d and %d", dev, there);
  }
  const EvictArgs a = {view(from), view(to), budget, recent, kept};
  cudaStream_t s = (cudaStream_t)stream;
  // CTAs per head: as many as have SMs of their own, as long as each has some thousand positions
  int cs = 1;
  while (cs < kCluster && heads * cs * 2 <= (size_t)sm_count(dev) && from->capacity > 4096 * cs) cs *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)heads * cs), cfg.blockDim = dim3(kSelect), cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cs, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
  if (int rc = check_launch("kv4 evict select", cfg.gridDim.x)) return rc;
  const int per = kThreads / (from->D / 16) * kMove;
  const unsigned nx = (unsigned)((budget + per - 1) / per);
  for (size_t h0 = 0; h0 < heads; h0 += 65535) {
    EvictArgs b = a;
    const size_t n = std::min<size_t>(65535, heads - h0);
    for (int i = 0; i < 2; ++i) {
      b.from.codes[i] += h0 * from->capacity * (from->D / 2), b.to.codes[i] += h0 * to->capacity * (to->D / 2);
      b.from.param[i] += h0 * from->capacity, b.to.param[i] += h0 * to->capacity;
    }
    b.from.weight += h0 * from->capacity, b.to.weight += h0 * to->capacity, b.kept += h0 * budget;
    const dim3 grid(nx, (unsigned)n);
    if (h0)  // behind another part of itself
      from->D == 64 ? evict_move_kernel<64><<<grid, kThreads, 0, s>>>(b) : evict_move_kernel<128><<<grid, kThreads, 0, s>>>(b);
    else
      launch_behind(from->D == 64 ? evict_move_kernel<64> : evict_move_kernel<128>, grid, kThreads, s, b);
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

// Whether the kernel for many rows (R per key/value head) is the faster one.  It begins with
// some 25 us more (128 decoded positions and 256 rows at a time), the other reads the
// cache once per 16 rows.  us of a call in a graph, bf16, this one and the other, at head dim 128 and at 64:
//   8 heads of 4000 positions   128 rows 41 and 32, 256 rows 46 and 52  |  128 rows 30 and 23, 256 rows 33 and 37
//   64 heads of 4000            32 rows 72 and 53, 64 rows 72 and 94, 128 rows 75 and 168  |  64 rows 64 and 66, 128 rows 64 and 116
//   8 heads of 30000            64 rows 80 and 67, 128 rows 82 and 115  |  64 rows 65 and 40, 128 rows 65 and 68
//   256 heads of 1000           64 rows 80 and 78, 128 rows 84 and 141  |  64 rows 69 and 40, 128 rows 69 and 73
// The line drawn goes by positions alone, between the head dims' and the shapes' own; it is farthest off for
// 64 rows over 64 heads of 4000 at head dim 128.  Positions are the capacity's, since lengths are known on the device
// only: a large cache that holds little takes the kernel that its capacity would need.
// With weights the other one also stores all scores and reads them back, this one computes them twice; up to 48
// rows that other one is the faster or about equal everywhere, with more it depends:
//   8 heads of 4000 positions   33 rows 55 and 45,  48 rows 56 and 48,  64 rows 56 and 68  |  48 rows 43 and 35, 64 rows 44 and 58
//   64 heads of 4000            33 rows 175 and 109, 48 rows 175 and 124, 64 rows 176 and 161  |  48 rows 153 and 89, 64 rows 153 and 118
//   8 heads of 30000            33 rows 174 and 98, 48 rows 174 and 117, 64 rows 175 and 151  |  48 rows 147 and 84, 64 rows 147 and 109
//   256 heads of 1000           33 rows 182 and 144, 48 rows 183 and 184, 64 rows 183 and 238  |  48 rows 160 and 141, 64 rows 159 and 184
static bool many_rows(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  const long long rows = (long long)Hq / c->H * N, passes = (rows + 15) / 16, positions = (long long)c->Z * c->H * c->capacity;
  return weights ? rows > kWeightRows : 2 * passes * positions > 800000 + 5 * positions;
}

static size_t attend_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  return many_rows(c, Hq, N, weights) ? prompt_workspace(c, Hq, N, weights) : rows_workspace(c, Hq, N, weights);
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
  const float scale_log2e = (float)(scale * 1.4426950408889634);
  if (!std::isfinite(scale_log2e)) return set_err(QFLASH_ERR_ARG, "kv4 attend: scale is not finite in fp32");
  if (cache->Z == 0) return QFLASH_OK;
  const size_t weight_bytes = (size_t)cache->Z * cache->H * cache->capacity * 4;
  if (weights_in && weights_in != cache->weight && overlap(weights_in, weight_bytes, cache->weight, weight_bytes))
    return set_err(QFLASH_ERR_ARG, "kv4 attend: weights_in overlaps the cache's weights");
  if (N == 0) {
    if (!weights_in || weights_in == cache->weight) return QFLASH_OK;
    OnDevice on(cache);
    if (on.rc) return on.rc;
    const int parts = std::min((cache->capacity + kThreads * 16 - 1) / (kThreads * 16), 1024);
    const unsigned grid = (unsigned)cache->Z * cache->H * parts;
    set_weights_kernel<<<grid, kThreads, 0, (cudaStream_t)stream>>>(view(cache), weights_in, parts);
    return check_launch("kv4 attend", grid);
  }
  if (!q || !out || !q_strides || !out_strides) return set_err(QFLASH_ERR_ARG, "kv4 attend: null pointer");
  if (q_strides[3] != 1 || out_strides[3] != 1) return set_err(QFLASH_ERR_ARG, "kv4 attend: innermost (head-dim) stride must be 1");
  const size_t need = attend_workspace(cache, Hq, N, weights_in != nullptr);
  if (!workspace || workspace_bytes < need)
    return set_err(QFLASH_ERR_ARG, "kv4 attend: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return set_err(QFLASH_ERR_ALIGN, "kv4 attend: workspace must be 16-byte aligned");
  OnDevice on(cache);
  if (on.rc) return on.rc;
  const int dev = on.dev;
  AttendArgs a;
  a.c = view(cache);
  a.q = q, a.out = out;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.os[i] = out_strides[i];
  a.rep = Hq / cache->H, a.N = N, a.new_lens = new_lens, a.causal = causal;
  a.scale_log2e = scale_log2e;
  a.weights_in = weights_in;
  return many_rows(cache, Hq, N, weights_in != nullptr) ? attend_prompt(a, dtype == kF16, workspace, dev, (cudaStream_t)stream)
                                 : attend_rows(a, dtype == kF16, workspace, dev, (cudaStream_t)stream);
}
