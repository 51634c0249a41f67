// Attention of many query rows over the 4-bit cache (prompts and their pieces):
// qflash_kv4_attend's path for launches that arithmetic bounds.
//
// Rows of a key/value head are numbered token by token, its rep query heads
// next to each other: row = token * rep + head, so that a tile of rows has one
// narrow range of causal limits and a key tile serves all heads of the group.
// A CTA holds 2 tiles of 128 rows and walks tiles of 128 keys:
//   4 warps decode: a thread owns a key, turns its codes into bf16 (or fp16)
//     numbers code - zero, exact, and writes them swizzled into shared memory;
//     scales go to a ring of their own, and stay outside of the products
//   1 warp issues tcgen05.mma: S = Q K^T into TMEM, O += P V with P from TMEM
//   2 x 4 warps do the softmax of a row tile each, a thread a row, and write P
//     over S.  The two tiles take turns: one's products run under the other's
//     softmax.
// P vs goes to the tensor cores as the sum of two bf16 terms (off by 2^-16), for the
// reasons given in the kernel for few rows; the second one costs bf16 queries 295 -> 355 us
// for the prompt's piece below.  A tile's P is formed against
// a reference from the tiles before it (at first the first tile's maximum), in one
// pass that takes 32 columns at a time and overwrites them: P above 1 costs no
// bits in floating point.  Where a tile's P add up to more than 2^16 the reference is
// raised for the next; only sums of 32 above 2^32 stop the pass, and what the tile has so
// far is scaled.  So the terms of an O are below 2^35 in all (2^34 of a tile that comes to that,
// less than 2^16 from each of the up to 2^17 tiles before it), and values below 2^92 cannot overflow it.
// The order of d within each 8 is 0 4 1 5 2 6 3 7 everywhere (codes d and d + 4
// of a word come out of one mask): Q is stored so, and the epilogue undoes it.
//
// Work split as in the kernel for few rows: tiles of all (sequence, row tile,
// head) units are numbered, each CTA takes an equal run, pieces of units are
// joined by a second kernel.
//
// Measured, prompt_kernel alone: 2048 tokens over 8000 positions, 8 heads x 4, head dim
// 128, bf16 (234 GFLOP) 355 us, 660 TFLOP/s, the tensor pipe active 46 % of the time; 4
// ragged prompts of up to 2049 tokens, 6 heads x 2, head dim 64, fp16 63 us.  A pair of
// tiles takes some 6700 cycles, of which its six products of 128 x 128 x 128 take 512 each (8192
// operations a cycle) and its 32768 exponentials 2048 (16 a cycle): what bounds it is the softmax
// warps' chain per 32 columns (TMEM load, exponentials, conversion, TMEM store) with one
// thread a row, and that products with V wait for the whole tile's P.  More instruction parallelism in
// the chain cost more than it gave.  With one term of P vs, 291 us then: chunks unrolled or
// two in turn 322 to 342 us, as the loops' instructions then outgrow their cache;
// 3 decoding warps 411; separate warps for K's and V's codes 361 to 387.
// ptxas spills 16 bytes of stores for head dim 128, and in prompt_weights_kernel 24 for 128 and 8 for 64.
//
// The attention weights need the rows' final maximum and sum, so a third kernel
// forms S^T = K Q^T again, keys in rows, and adds up exp(S - m) / l along its
// columns in a fixed order: no atomics.
#include <algorithm>
#include <atomic>

#include "kv4_common.cuh"
#include "sm100_ptx.cuh"

namespace qfb {
namespace kv4 {

constexpr int kM = 128;           // rows of a tile, TMEM lanes
constexpr int kKeys = 128;        // keys of a tile
constexpr int kRows = 2 * kM;     // rows of a CTA
constexpr int kRing = 4;          // tiles of scales
constexpr int kPrompt = 512;      // threads: 8 warps of softmax, 4 that decode, 1 that issues products, 3 idle

struct PromptArgs {
  AttendArgs a;
  int rows, row_tiles;  // N * rep, and that over 256
  int grid;
  bool vec_q, vec_o;
  uint32_t magic_k, magic_v;
  float* parts;   // [grid][2][256 (D + 2)]
  float2* stats;  // [Z H][rows]: maximum (log2 units) and 1 / sum; null without weights
};

// kind::f16 instruction descriptor, fp32 accumulator: [4,6) D format 1 = f32,
// [7,10) and [10,13) A and B format (0 f16, 1 bf16), [16] B major (1 = MN),
// [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t idesc_f16(int N, bool bf16, bool b_mn_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
// Issued by the lane with `on`, which all lanes of a warp reach together: in a branch of one
// lane's every descriptor would be moved to the uniform registers by itself.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t on) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t on) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
               : "memory");
}
// The same value in all lanes, known to be.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }
__device__ __forceinline__ void tmem_ld32f(uint32_t addr, float* r) {
  int v[32];
  tmem_ld32(addr, v);
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __int_as_float(v[i]);
}
// 32 lanes x 32 columns of 32 bits, begun; the registers hold them after tmem_arrived.
__device__ __forceinline__ void tmem_begin32(uint32_t addr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_arrived(float (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                 "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               :);
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
               "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}
// pairs of fp32, one instruction for two
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
// a, b = a * x + s, b * y + t
__device__ __forceinline__ void fma2(float& a, float& b, float x, float y, float s, float t) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y), "f"(s), "f"(t));
}

// Waits with a limit; after it (or another warp's) every role leaves its loops.
struct Waiter {
  volatile uint32_t* abort;
  int32_t* ctl;
  // A warp's lanes wait together and get the same answer.
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    bool there = mbar_try_wait(bar, parity);
    if (__all_sync(~0u, there)) return true;
    const long long t0 = clock64();
    while (!there) {
      there = mbar_try_wait_hint(bar, parity, 100000);
      if (there || *abort) break;
      if (clock64() - t0 > kWaitCycles) {
        *abort = 1;
        atomicOr(&ctl[1], 2);
        break;
      }
    }
    return __all_sync(~0u, there);
  }
};

// 8 codes as 4 words of two numbers code - zero, in the order 0 4, 1 5, 2 6, 3 7:
// set into the mantissa of `magic`, 128 (bf16) or 1024 (fp16), which is a kernel
// argument because lop3 takes one immediate and the mask is it.
template <bool FP16>
__device__ __forceinline__ uint4 decode8(uint32_t w, uint32_t magic, uint32_t zero) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(magic));  // (w & mask) | magic
    if (FP16)
      asm("sub.f16x2 %0, %1, %2;" : "=r"(y[i]) : "r"(m), "r"(zero));
    else
      asm("sub.bf16x2 %0, %1, %2;" : "=r"(y[i]) : "r"(m), "r"(zero));
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}
template <bool FP16>
__device__ __forceinline__ uint32_t zero_pair(uint32_t param) {
  if (FP16) {
    const __half2 x = __float2half2_rn(1024.f + param_zero(param));
    return *reinterpret_cast<const uint32_t*>(&x);
  }
  return pack_bf16(128.f + param_zero(param), 128.f + param_zero(param));
}

// One vector's codes, decoded, as row `row` of a 128-row tile in shared memory:
// blocks of 64 elements (128 bytes, swizzled by 16-byte chunks over 8 rows).
// A compact loop that takes codes[0] and rotates them: the warps of a CTA do
// different things, and together they must not outgrow the instruction caches.
template <int D, bool FP16>
__device__ __forceinline__ void put_codes(uint32_t base, int row, uint4 (&codes)[D / 32], uint32_t magic, uint32_t zero) {
  const uint32_t to = base + row * 128, turn = (uint32_t)(row & 7) << 4;
#pragma unroll 1
  for (int i = 0; i < D / 32; ++i) {
    const uint32_t w[4] = {codes[0].x, codes[0].y, codes[0].z, codes[0].w};
    const uint32_t block = to + (i >> 1) * (128 * 128), chunk = (i & 1) * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) sts128(block + ((chunk + 16 * j) ^ turn), decode8<FP16>(w[j], magic, zero));
#pragma unroll
    for (int e = 0; e + 1 < D / 32; ++e) codes[e] = codes[e + 1];
  }
}
// The same in the elements' own order: an exchange of halves more per word.
template <int D, bool FP16>
__device__ __forceinline__ void put_codes_plain(uint32_t base, int row, uint4 (&codes)[D / 32], uint32_t magic, uint32_t zero) {
  const uint32_t to = base + row * 128, turn = (uint32_t)(row & 7) << 4;
#pragma unroll 1
  for (int i = 0; i < D / 32; ++i) {
    const uint32_t w[4] = {codes[0].x, codes[0].y, codes[0].z, codes[0].w};
    const uint32_t block = to + (i >> 1) * (128 * 128), chunk = (i & 1) * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 y = decode8<FP16>(w[j], magic, zero);  // 0 4, 1 5, 2 6, 3 7
      sts128(block + ((chunk + 16 * j) ^ turn), make_uint4(__byte_perm(y.x, y.y, 0x5410), __byte_perm(y.z, y.w, 0x5410),
                                                           __byte_perm(y.x, y.y, 0x7632), __byte_perm(y.z, y.w, 0x7632)));
    }
#pragma unroll
    for (int e = 0; e + 1 < D / 32; ++e) codes[e] = codes[e + 1];
  }
}
// One query row in its own order, copied past the registers where it starts on a
// 16-byte boundary (complete after the copies' wait), zeros for one that is not there.
template <int D>
__device__ __forceinline__ void copy_query(uint32_t base, int row, const uint16_t* q, const uint16_t* any, bool vec) {
#pragma unroll 4
  for (int chunk = 0; chunk < D / 8; ++chunk) {
    const uint32_t to = base + (chunk / 8) * (128 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
    if (vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(q ? q + 8 * chunk : any), "r"(q ? 16 : 0) : "memory");
    } else {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (q) {
        const uint16_t* p = q + 8 * chunk;
        x = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
      }
      sts128(to, x);
    }
  }
}
// One query row in the order of put_codes.
template <int D>
__device__ __forceinline__ void put_query(uint32_t base, int row, const uint16_t* q, bool vec) {
#pragma unroll 4
  for (int chunk = 0; chunk < D / 8; ++chunk) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (q) {
      if (vec) {
        x = __ldg(reinterpret_cast<const uint4*>(q) + chunk);
      } else {
        const uint16_t* p = q + 8 * chunk;
        x = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
      }
    }
    sts128(base + (chunk / 8) * (128 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4),
           make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                      __byte_perm(x.y, x.w, 0x7632)));
  }
}
// Shared-memory descriptors, from the low word of the tile's: one thread issues all
// products, and forming 64-bit descriptors step by step cost it more time than
// the products take.  K-major operand (Q, K): a step of 16 elements is 32 bytes in a
// block of 64 elements; MN-major operand (V): a step of 16 keys is 16 rows of 128 bytes.
__device__ __forceinline__ uint32_t k_word(uint32_t base) { return (uint32_t)smem_desc(base, 16, 1024, kSw128); }
__device__ __forceinline__ uint32_t mn_word(uint32_t base) { return (uint32_t)smem_desc(base, 128 * 128, 1024, kSw128); }
__device__ __forceinline__ uint64_t desc_of(uint32_t word) {
  constexpr uint32_t kHigh = (uint32_t)(smem_desc(0, 0, 1024, kSw128) >> 32);
  return (uint64_t)kHigh << 32 | word;
}
__device__ __forceinline__ uint64_t k_desc(uint32_t word, int step) { return desc_of(word + (step >> 2) * (128 * 128 / 16) + (step & 3) * 2); }
__device__ __forceinline__ uint64_t mn_desc(uint32_t word, int step) { return desc_of(word + step * (16 * 128 / 16)); }

// P's column for a step of 16 keys: 32 keys' first terms lie in the first 16 of their scores' 32 columns, the
// second terms behind them.
__device__ __forceinline__ constexpr uint32_t p_col(int step) { return 32 * (step >> 1) + 8 * (step & 1); }

// ------------------------------------------------------------------ work split
// Key tiles of row tile rt of sequence z.
__device__ __forceinline__ int unit_tiles(const PromptArgs& p, int z, int rt) {
  const AttendArgs& a = p.a;
  const Span sp = span_of(a, z);
  const int first = rt * kRows / a.rep, last = min(min(a.N, sp.fresh), (rt * kRows + kRows - 1) / a.rep + 1);
  return first >= last ? 0 : (sp.limit(a, last - 1) + kKeys - 1) / kKeys;
}

// Where a CTA is in its run.  All lanes of a warp hold the same.
struct Walk {
  int z, rt, h, tiles;   // the unit
  long long first;       // where it begins: kBegin places, then its tiles
  long long at, stop;    // the run
  int t0, t1;            // the piece: key tiles of the unit
  int places;            // what of the run it takes
  bool whole;

  __device__ __forceinline__ void cut() {
    const int u0 = (int)(at - first), u1 = (int)min((long long)cost_of(tiles), u0 + (stop - at));
    places = u1 - u0;
    t0 = max(0, u0 - kBegin);
    t1 = max(0, u1 - kBegin);
    whole = t0 == 0 && t1 == tiles;
  }
  // The unit that holds a place.  One warp together.
  __device__ __forceinline__ bool seek(const PromptArgs& p, long long where) {
    const int lane = threadIdx.x & 31, n = p.a.c.Z * p.row_tiles, H = p.a.c.H;
    long long base = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const int t = i < n ? unit_tiles(p, i / p.row_tiles, i % p.row_tiles) : 0;
      const long long mine = (long long)cost_of(t) * H;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned hit = __ballot_sync(~0u, where >= base + sum - mine && where < base + sum);
      if (hit) {
        const int l = __ffs(hit) - 1;
        tiles = __shfl_sync(~0u, t, l);
        first = base + __shfl_sync(~0u, sum - mine, l);
        z = (i0 + l) / p.row_tiles, rt = (i0 + l) % p.row_tiles;
        h = (int)((where - first) / cost_of(tiles));
        first += (long long)h * cost_of(tiles);
        return true;
      }
      base += __shfl_sync(~0u, sum, 31);
    }
    return false;
  }
  __device__ static long long total_cost(const PromptArgs& p) {
    const int lane = threadIdx.x & 31, n = p.a.c.Z * p.row_tiles;
    long long sum = 0;
    for (int i = lane; i < n; i += 32) sum += cost_of(unit_tiles(p, i / p.row_tiles, i % p.row_tiles));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    return sum * p.a.c.H;
  }
  // The run's first piece with tiles in it, from `at` on.  One warp together.
  __device__ __forceinline__ bool begin(const PromptArgs& p) {
    if (!seek(p, at)) return false;  // only if lens changed meanwhile
    cut();
    return t1 > t0 || next(p);
  }
  // On to the run's next piece with tiles in it; false behind its end.
  __device__ __forceinline__ bool next(const PromptArgs& p) {
    do {
      at += places;
      if (at >= stop) return false;
      first += cost_of(tiles);
      if (++h == p.a.c.H) {
        h = 0;
        do {
          if (++rt == p.row_tiles) {
            rt = 0;
            if (++z >= p.a.c.Z) return false;  // only if lens changed meanwhile
          }
          tiles = unit_tiles(p, z, rt);
        } while (tiles == 0);
      }
      cut();
    } while (t1 <= t0);
    return true;
  }
};
__device__ __forceinline__ long long run_begin(long long total, int grid, int cta) { return total * cta / grid; }

// ------------------------------------------------------------------ attention
template <int D>
struct Layout {
  static constexpr uint32_t TILE = 128 * D * 2;
  static constexpr uint32_t Q = 0, K = 2 * TILE, V = 4 * TILE, KS = 6 * TILE, VS = KS + kRing * 512, BARS = VS + kRing * 512;
  static constexpr uint32_t BYTES = BARS + 256 + 1024;  // with room to align the base
};

// A row of the softmax, held by one thread: the reference of its exponentials
// (log2), their sum, and what O has yet to be multiplied by.
struct RowState {
  float m, l, late;
};

// O times f.  The last product into it is done: this tile's scores were committed after that.
template <int D>
__device__ __forceinline__ void scale_out(uint32_t o_at, float f) {
#pragma unroll 1
  for (int q = 0; q < D / 32; ++q) {
    int o[32];
    tmem_ld32(o_at + 32 * q, o);
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_int(__int_as_float(o[i]) * f);
    tmem_st32(o_at + 32 * q, o);
  }
}

// 32 scores against a row's reference; those from `lim` on (of the tile's 128) masked.
template <bool FULL>
__device__ __forceinline__ void differences(uint32_t s_at, const float4* ks, int q, int lim, float neg, float (&x)[32]) {
  tmem_begin32(s_at + 32 * q, x);
  tmem_arrived(x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 f = ks[8 * q + i];
    fma2(x[4 * i], x[4 * i + 1], f.x, f.y, neg, neg);
    fma2(x[4 * i + 2], x[4 * i + 3], f.z, f.w, neg, neg);
  }
  if (!FULL) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (32 * q + i >= lim) x[i] = -INFINITY;
  }
}
__device__ __forceinline__ float largest(const float (&x)[32]) {
  float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; i += 2) a[i / 2 & 3] = max3(a[i / 2 & 3], x[i], x[i + 1]);
  return fmaxf(max3(a[0], a[1], a[2]), a[3]);
}
// The first tile's own maximum is the reference to begin with.
__device__ __noinline__ float first_reference(uint32_t s_at, const float4* ks, int lim) {
  float m = -INFINITY;
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    float x[32];
    differences<false>(s_at, ks, q, lim, 0.f, x);
    m = fmaxf(m, largest(x));
  }
  return m;
}
// Raises the reference of rows for which chunk q is `high` to the chunk's maximum,
// by a whole number (or from nothing to the first score), and scales O and the P of
// this tile's chunks before q.  Returns the reference and what the sums are to be
// multiplied by.  Out of line, as its registers would burden every tile's loop.
template <int D>
__device__ __noinline__ float2 raise_reference(float m, uint32_t s_at, uint32_t o_at, const float4* ks, int q, int lim,
                                               bool high, bool first) {
  float x[32];
  differences<false>(s_at, ks, q, lim, m == -INFINITY ? 0.f : -m, x);
  const float top = largest(x);
  const bool up = high && top > (m == -INFINITY ? -INFINITY : 0.f);
  const float by = !up ? 0.f : m == -INFINITY ? top : ceilf(top);
  const float f = !up ? 1.f : m == -INFINITY ? 0.f : ex2(-by);
  m = !up ? m : m == -INFINITY ? top : m + by;
  if (!first) scale_out<D>(o_at, f);
  tmem_wait_st();
  const uint32_t ff = pack_bf16(f, f);
#pragma unroll 1
  for (int e = 0; e < 2 * q; ++e) {
    uint32_t y[16];
    const uint32_t at = s_at + 16 * e;
    tmem_ld16(at, y);
#pragma unroll
    for (int i = 0; i < 16; ++i) asm("mul.bf16x2 %0, %0, %1;" : "+r"(y[i]) : "r"(ff));
    tmem_st16(at, y);
  }
  return make_float2(m, f);
}

// One tile of 128 scores of a row: P over the scores.  FULL: the row sees all of
// them, else the first `lim`.  All steps are written over many independent
// elements: a warp's latencies, not its instructions, are what it waits for.
// For the same reason no maximum stands before the exponentials: their sum says
// afterwards, before P is stored, whether the reference is still good enough, and
// what it has to become.
template <int D, bool FULL>
__device__ __forceinline__ void softmax_tile(RowState& r, uint32_t s_at, uint32_t o_at, const float4* ks, const float4* vs,
                                             int lim, bool first) {
  if (first) {
    r.m = first_reference(s_at, ks, lim);
  } else if (__any_sync(~0u, r.late != 1.f)) {
    scale_out<D>(o_at, r.late);
    r.late = 1.f;
  }
  float total = 0.f;
  bool raised = false;
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    float x[32];
    differences<FULL>(s_at, ks, q, lim, r.m == -INFINITY ? 0.f : -r.m, x);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = ex2(x[i]);
    float c[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; i += 2) add2(c[i & 6], c[(i & 6) + 1], x[i], x[i + 1]);
    add2(c[0], c[1], c[2], c[3]);
    add2(c[4], c[5], c[6], c[7]);
    add2(c[0], c[1], c[4], c[5]);
    const float sum = c[0] + c[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 f = vs[8 * q + i];
      mul2(x[4 * i], x[4 * i + 1], f.x, f.y);
      mul2(x[4 * i + 2], x[4 * i + 3], f.z, f.w);
    }
    if (!FULL) {  // a masked position's scale may be anything
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (32 * q + i >= lim) x[i] = 0.f;
    }
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) hi[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      add2(x[2 * i], x[2 * i + 1], -__uint_as_float(hi[i] << 16), -__uint_as_float(hi[i] & 0xffff0000u));
      lo[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    }
    // Too large to go on with (or, for a row without a score above -inf so far, not to be judged by the sum):
    // the chunk again, against a higher reference.  Asked only here, so that nothing above waits for the answer.
    const bool high = !raised && (sum > 4294967296.f || (r.m == -INFINITY && lim > 32 * q));  // 2^32
    if (__any_sync(~0u, high)) {
      const float2 up = raise_reference<D>(r.m, s_at, o_at, ks, q, lim, high, first);
      r.m = up.x;
      r.l *= up.y, total *= up.y;
      raised = true;
      --q;
      continue;
    }
    raised = false;
    total += sum;
    tmem_st16(s_at + 32 * q, hi);
    tmem_st16(s_at + 32 * q + 16, lo);
  }
  r.l += total;
  tmem_wait_st();
  // The tile's sum is its largest P up to a factor of 128: a reference raised to it leaves that 2^-7 at least.
  if (total > 65536.f && total < INFINITY) {
    const float by = (float)((int)(__float_as_uint(total) >> 23) - 127), f = ex2(-by);
    r.m += by;
    r.l *= f, r.late *= f;
  }
}

template <int D, bool FP16>
__global__ void __launch_bounds__(kPrompt, 1) prompt_kernel(PromptArgs p) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  const uint32_t bars = base + L::BARS;
  auto k_full = [&](int i) { return bars + 8 * i; };
  auto k_empty = [&](int i) { return bars + 16 + 8 * i; };
  auto v_full = [&](int i) { return bars + 32 + 8 * i; };
  auto v_empty = [&](int i) { return bars + 48 + 8 * i; };
  auto q_full = [&](int t) { return bars + 64 + 8 * t; };
  auto s_full = [&](int t) { return bars + 80 + 8 * t; };
  auto p_full = [&](int t) { return bars + 96 + 8 * t; };
  auto o_full = [&](int t) { return bars + 112 + 8 * t; };
  const uint32_t done = bars + 128, slot = bars + 136;
  volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(smem + L::BARS + 140);
  float* const ks_ring = reinterpret_cast<float*>(smem + L::KS);
  float* const vs_ring = reinterpret_cast<float*>(smem + L::VS);

  if (warp == 12) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {  // arrivals: one per warp that writes
        mbar_init(k_full(i), 4), mbar_init(v_full(i), 4);
        mbar_init(k_empty(i), 1), mbar_init(v_empty(i), 1);
        mbar_init(q_full(i), 4), mbar_init(p_full(i), 4);
        mbar_init(s_full(i), 2), mbar_init(o_full(i), 1);
      }
      mbar_init(done, 1);
      *abort = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem = 0;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  const Waiter wait{abort, c.ctl};
  auto warp_arrive = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };

  may_begin();
  Walk w;
  const long long total = Walk::total_cost(p);
  const int grid = (int)min((long long)p.grid, total);
  bool any = (int)blockIdx.x < grid;
  if (any) {
    w.at = run_begin(total, grid, blockIdx.x);
    w.stop = run_begin(total, grid, blockIdx.x + 1);
    any = w.begin(p);
  }

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    const int t = warp >> 2, lrow = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
    uint32_t n = 0, pieces = 0;  // key tiles and pieces so far
    // this thread's row of a unit: queries into shared memory
    auto bring_query = [&] {
      const Span sp = span_of(a, w.z);
      const int row = w.rt * kRows + t * kM + lrow, tok = row / a.rep, head = w.h * a.rep + row % a.rep;
      const bool live = row < p.rows && tok < sp.fresh;
      put_query<D>(base + L::Q + t * L::TILE, lrow,
                   live ? (const uint16_t*)a.q + (w.z * a.qs[0] + head * a.qs[1] + tok * a.qs[2]) : nullptr, p.vec_q);
      fence_proxy_async_smem();
      warp_arrive(q_full(t));
    };
    if (any) bring_query();
    while (any) {
      const Span sp = span_of(a, w.z);
      const int row = w.rt * kRows + t * kM + lrow, tok = row / a.rep, head = w.h * a.rep + row % a.rep;
      const int limit = row < p.rows && tok < sp.fresh ? sp.limit(a, tok) : 0;
      const bool whole = w.whole;
      const int z = w.z, h = w.h;
      RowState r = {-INFINITY, 0.f, 1.f};
      for (int j = w.t0; j < w.t1; ++j, ++n) {
        if (!wait(s_full(t), n & 1)) goto out;
        tc_fence_after();
        const float4* ks = reinterpret_cast<const float4*>(ks_ring + (n & (kRing - 1)) * kKeys);
        const float4* vs = reinterpret_cast<const float4*>(vs_ring + (n & (kRing - 1)) * kKeys);
        const int lim = limit - j * kKeys;
        if (__all_sync(~0u, lim >= kKeys))
          softmax_tile<D, true>(r, s_at, o_at, ks, vs, lim, j == w.t0);
        else
          softmax_tile<D, false>(r, s_at, o_at, ks, vs, lim, j == w.t0);
        tc_fence_before();
        warp_arrive(p_full(t));
      }
      // the last scores are made, so the next unit's queries may come: their products with the first keys run
      // under this unit's output
      any = w.next(p);
      if (any) bring_query();
      if (!wait(o_full(t), pieces & 1)) goto out;
      tc_fence_after();
      {
        const float inv = 1.f / r.l;
        const bool write = row < p.rows;
        float* part = p.parts + ((size_t)blockIdx.x * 2 + (pieces ? 1 : 0)) * (kRows * (D + 2));
        const size_t to = z * a.os[0] + head * a.os[1] + (size_t)tok * a.os[2];
        if (write) {
          if (!whole)
            part[t * kM + lrow] = r.m, part[kRows + t * kM + lrow] = r.l;
          else if (p.stats)
            p.stats[((size_t)z * c.H + h) * p.rows + row] = make_float2(r.m, inv);
        }
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          float o[32];
          tmem_ld32f(o_at + 32 * q, o);
          if (!write) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= r.late;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float y[8] = {o[8 * g], o[8 * g + 2], o[8 * g + 4], o[8 * g + 6], o[8 * g + 1], o[8 * g + 3], o[8 * g + 5], o[8 * g + 7]};
            if (whole) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = limit > 0 ? y[e] * inv : 0.f;
              if (FP16)
                store8((__half*)a.out + to + 32 * q + 8 * g, p.vec_o, x);
              else
                store8((__nv_bfloat16*)a.out + to + 32 * q + 8 * g, p.vec_o, x);
            } else {
              store8(part + 2 * kRows + (t * kM + lrow) * D + 32 * q + 8 * g, true, y);
            }
          }
        }
        tc_fence_before();
      }
      ++pieces;
    }
  } else if (warp < 12) {
    // ---------------------------------------------------------------- decoding
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int key = tid - 256;
    uint32_t n = 0;
    while (any) {
      const size_t head = ((size_t)w.z * c.H + w.h) * c.C;
      const int len = length_of(c, w.z);
      for (int j = w.t0; j < w.t1; ++j, ++n) {
        const int pos = j * kKeys + key, at = max(0, min(pos, len - 1));
        const uint32_t kp = pos < len ? __ldg(c.param[0] + head + at) : 0u, vp = pos < len ? __ldg(c.param[1] + head + at) : 0u;
        uint4 kc[D / 32], vc[D / 32];
        const uint4* src = reinterpret_cast<const uint4*>(c.codes[0] + (head + at) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) kc[i] = __ldg(src + i);
        src = reinterpret_cast<const uint4*>(c.codes[1] + (head + at) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) vc[i] = __ldg(src + i);
        const int st = n & 1, ring = (n & (kRing - 1)) * kKeys;
        if (!wait(k_empty(st), (n >> 1 & 1) ^ 1)) goto out;
        // this slot's last tile is 4 back: the products of the tile 2 back, which k_empty waited for, came after its softmax
        ks_ring[ring + key] = param_scale(kp) * a.scale_log2e;
        vs_ring[ring + key] = param_scale(vp);
        put_codes<D, FP16>(base + L::K + st * L::TILE, key, kc, p.magic_k, zero_pair<FP16>(kp));
        fence_proxy_async_smem();
        warp_arrive(k_full(st));
        if (!wait(v_empty(st), (n >> 1 & 1) ^ 1)) goto out;
        put_codes<D, false>(base + L::V + st * L::TILE, key, vc, p.magic_v, zero_pair<false>(vp));
        fence_proxy_async_smem();
        warp_arrive(v_full(st));
      }
      any = w.next(p);
    }
  } else {
    // ---------------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 12) {
      constexpr uint32_t IS = idesc_f16(kKeys, !FP16, false), IO = idesc_f16(D, true, true);
      const uint32_t q_word = k_word(base + L::Q), kk_word = k_word(base + L::K), v_word = mn_word(base + L::V);
      uint32_t n = 0, pieces = 0;
      // S = Q K^T of row tile t and key tile g
      auto scores = [&](int t, uint32_t g) {
        const uint32_t kw = uniform(kk_word + (g & 1) * (L::TILE / 16)), qw = uniform(q_word + t * (L::TILE / 16)), to = uniform(tmem + t * 128);
#pragma unroll 1
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            mma_ss(to, k_desc(qw + b * 1024, s), k_desc(kw + b * 1024, s), IS, s > 0 ? 1 : b, lane == 0);
        if (lane == 0) {
          tc_commit(s_full(t));
          mbar_arrive(s_full(t));  // passes on the scales that k_full's wait made visible here
        }
        __syncwarp();
      };
      while (any) {
        const int tiles = w.t1 - w.t0;
        if (!wait(k_full(n & 1), n >> 1 & 1)) goto out;
        for (int t = 0; t < 2; ++t) {
          if (!wait(q_full(t), pieces & 1)) goto out;
          tc_fence_after();
          scores(t, n);
        }
        if (lane == 0) tc_commit(k_empty(n & 1));
        __syncwarp();
        for (int j = 0; j < tiles; ++j, ++n) {
          // first what is there long before P, so that nothing stands between P and its products
          if (!wait(v_full(n & 1), n >> 1 & 1)) goto out;
          if (j + 1 < tiles && !wait(k_full((n + 1) & 1), (n + 1) >> 1 & 1)) goto out;
          for (int t = 0; t < 2; ++t) {
            if (!wait(p_full(t), n & 1)) goto out;
            tc_fence_after();
            const uint32_t vw = uniform(v_word + (n & 1) * (L::TILE / 16)), to = uniform(tmem + 256 + t * 128), from = uniform(tmem + t * 128);
            const uint32_t more = uniform(j > 0);
#pragma unroll 1
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                mma_ts(to, from + 64 * b + p_col(s), mn_desc(vw + 512 * b, s), IO, s > 0 ? 1 : more | b, lane == 0);
                mma_ts(to, from + 64 * b + 16 + p_col(s), mn_desc(vw + 512 * b, s), IO, 1, lane == 0);
              }
            if (j + 1 < tiles) {
              scores(t, n + 1);
            } else {
              if (lane == 0) tc_commit(o_full(t));
              __syncwarp();
            }
            if (t == 1) {
              // Both row tiles are through with this tile's values and the next one's keys when these are.
              if (lane == 0) {
                tc_commit(v_empty(n & 1));
                if (j + 1 < tiles) tc_commit(k_empty((n + 1) & 1));
              }
              __syncwarp();
            }
          }
        }
        ++pieces;
        any = w.next(p);
      }
    }
  }
out:
  __syncwarp();
  if (warp == 12) {  // nothing of this CTA's may be under way when its TMEM goes
    if (lane == 0) tc_commit(done);
    __syncwarp();
    mbar_wait(done, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// Adds about 10 us to a call (reading the pieces back, 32 rows a block for parallel loads).
// Joins units that several CTAs held: blockIdx.x < 8 grid: 32 rows of the unit that
// run blockIdx.x / 8's beginning is the first to cut; the others write the
// zeros of units with nothing to see.
template <int D, bool FP16>
__global__ void __launch_bounds__(256) prompt_finish_kernel(PromptArgs p) {
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  constexpr int kPart = kRows * (D + 2);
  // one block at least waits, whatever it has to do: the kernels behind this one go by its end
  if (blockIdx.x == 0) wait_for_previous();
  auto put = [&](int z, int h, int row, int col, const float (&x)[8]) {
    const int tok = row / a.rep;
    const size_t to = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + (size_t)tok * a.os[2] + col;
    if (FP16)
      store8((__half*)a.out + to, p.vec_o, x);
    else
      store8((__nv_bfloat16*)a.out + to, p.vec_o, x);
  };
  if ((int)blockIdx.x >= 8 * p.grid) {
    const int i = blockIdx.x - 8 * p.grid, z = i / p.row_tiles, rt = i % p.row_tiles;
    if (unit_tiles(p, z, rt) > 0) return;
    wait_for_previous();
    const float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int e = threadIdx.x; e < kRows * (D / 8); e += 256) {
      const int row = rt * kRows + e / (D / 8);
      if (row < p.rows)
        for (int h = 0; h < c.H; ++h) put(z, h, row, e % (D / 8) * 8, x);
    }
    return;
  }
  const int k = blockIdx.x / 8;
  const long long total = Walk::total_cost(p);
  const int grid = (int)min((long long)p.grid, total);
  if (k == 0 || k >= grid) return;
  Walk w;
  const long long cut = run_begin(total, grid, k);
  // a cut that has tiles of its unit before it, and is the first to
  if (!w.seek(p, cut) || cut <= w.first + kBegin || run_begin(total, grid, k - 1) > w.first + kBegin) return;
  const long long end = w.first + cost_of(w.tiles);
  const Span sp = span_of(a, w.z);
  const int first = run_begin(total, grid, k - 1) < w.first ? 2 * (k - 1) + 1 : 2 * (k - 1);
  wait_for_previous();
  for (int e = threadIdx.x; e < 32 * (D / 8); e += 256) {
    const int r = (blockIdx.x & 7) * 32 + e / (D / 8), col = e % (D / 8) * 8, row = w.rt * kRows + r;
    if (row >= p.rows) break;
    const float* part = p.parts + (size_t)first * kPart;
    float m = part[r], l = part[kRows + r], o[8];
    read8(part + 2 * kRows + r * D + col, o);
    for (int q = k; q < grid && run_begin(total, grid, q) < end; ++q) {
      part = p.parts + (size_t)2 * q * kPart;
      const float pm = part[r], pl = part[kRows + r], mx = fmaxf(m, pm);
      const float f0 = m == -INFINITY ? 1.f : ex2(m - mx), f1 = pm == -INFINITY ? 1.f : ex2(pm - mx);
      float x[8];
      read8(part + 2 * kRows + r * D + col, x);
      l = l * f0 + pl * f1;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = o[i] * f0 + x[i] * f1;
      m = mx;
    }
    const int tok = row / a.rep;
    const bool seen = tok < sp.fresh && sp.limit(a, tok) > 0;
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = seen ? o[i] * inv : 0.f;
    put(w.z, w.h, row, col, o);
    if (p.stats && col == 0) p.stats[((size_t)w.z * c.H + w.h) * p.rows + row] = make_float2(m, inv);
  }
}

// ------------------------------------------------------------------ weights
constexpr int kWeigh = 416;
template <int D>
struct WLayout {
  static constexpr uint32_t TILE = 128 * D * 2;
  // query tiles: 3 where two CTAs' fit into an SM
  static constexpr int COUNT = D == 64 ? 3 : 2;
  static constexpr uint32_t K = 0, Q = TILE, COL = (1 + COUNT) * TILE, BARS = COL + COUNT * 3 * 512;
  static constexpr uint32_t BYTES = BARS + 128 + 1024;
};

// Two CTAs (a cluster) per 128 positions of a head, with every other row tile each,
// as the first positions of a prompt are seen by all its rows, one tile after
// the other.  Warps 0-7 add up (two threads a position, for 64 columns of a tile
// each), warps 8-11 bring query tiles, warp 12 issues the products.  Bound by the
// chain from TMEM load to exponentials and sums; the 4 ragged prompts above take 42 us, with one CTA for 128 positions 57,
// and with two query tiles in flight as well 80.
template <int D, bool FP16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWeigh, 2) prompt_weights_kernel(PromptArgs p) {
  using L = WLayout<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  // the first positions first: with a causal limit most rows see them
  const int rank = (int)cluster_rank(), unit = blockIdx.x / 2;
  const int heads = c.Z * c.H, zh = unit % heads, key0 = unit / heads * kKeys, z = zh / c.H, h = zh % c.H;
  const Span sp = span_of(a, z);
  if (key0 >= sp.len) return;  // both CTAs together, here and below
  // rows that see position key0: from token `first` on
  const int first = a.causal ? max(0, key0 - (sp.len - sp.fresh)) : 0;
  const int rt0 = first < sp.fresh ? first * a.rep / kM : 0, rt1 = first < sp.fresh ? (sp.fresh * a.rep + kM - 1) / kM : 0;
  const size_t head = (size_t)zh * c.C;
  if (rt0 >= rt1) {
    const int key = key0 + tid;
    if (rank == 0 && tid < kKeys && key < sp.len) c.weight[head + key] = a.weights_in[head + key];
    return;
  }
  const int tiles = max(0, (rt1 - rt0 - rank + 1) / 2);  // this CTA's: rt0 + rank, and every second from there on
  const uint32_t bars = base + L::BARS;
  auto q_full = [&](int i) { return bars + 8 * i; };
  auto q_empty = [&](int i) { return bars + 24 + 8 * i; };
  auto s_full = [&](int i) { return bars + 48 + 8 * i; };
  auto s_empty = [&](int i) { return bars + 64 + 8 * i; };
  const uint32_t k_full = bars + 80, done = bars + 88, slot = bars + 96;
  volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(smem + L::BARS + 100);
  __shared__ float other[kKeys];
  float* const col = reinterpret_cast<float*>(smem + L::COL);  // [2][3][128]: maximum, 1 / sum, limit
  if (warp == 12) {
    if (lane == 0) {
      for (int i = 0; i < L::COUNT; ++i) mbar_init(q_full(i), 4), mbar_init(q_empty(i), 9);
      for (int i = 0; i < 2; ++i) mbar_init(s_full(i), 1), mbar_init(s_empty(i), 8);
      mbar_init(k_full, 4), mbar_init(done, 1);
      *abort = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem = 0;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  const Waiter wait{abort, c.ctl};

  auto warp_arrive = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  const int key = key0 + (tid & 127);
  float sum0 = 0.f, sum1 = 0.f;
  if (warp < 8) {
    const int at = min(key, sp.len - 1), half = warp >> 2;
    const uint32_t kp = key < sp.len ? __ldg(c.param[0] + head + at) : 0u;
    const float ks = param_scale(kp) * a.scale_log2e;
    if (half == 0) {
      uint4 kc[D / 32];
      const uint4* src = reinterpret_cast<const uint4*>(c.codes[0] + (head + at) * (D / 2));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) kc[i] = __ldg(src + i);
      put_codes_plain<D, FP16>(base + L::K, tid, kc, p.magic_k, zero_pair<FP16>(kp));
      fence_proxy_async_smem();
      warp_arrive(k_full);
    }
    const uint32_t s_at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 64 * half;
    for (int g = 0; g < tiles; ++g) {
      const int rt = rt0 + rank + 2 * g, b = g & 1, qb = g % L::COUNT;
      if (!wait(s_full(b), g >> 1 & 1) || !wait(q_full(qb), g / L::COUNT & 1)) goto out;
      tc_fence_after();
      const float4* cm = reinterpret_cast<const float4*>(col + qb * 384) + 16 * half;
      const float4* ci = cm + 32;
      const int4* cl = reinterpret_cast<const int4*>(cm + 64);
      // every row of the tile is there and sees all 128 positions
      const bool full = (rt + 1) * kM <= sp.fresh * a.rep && sp.limit(a, rt * kM / a.rep) >= key0 + kKeys;
#pragma unroll 1
      for (int q = 0; q < 2; ++q) {
        float x[32];
        tmem_begin32(s_at + b * 128 + 32 * q, x);
        tmem_arrived(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 m = cm[8 * q + i];
          fma2(x[4 * i], x[4 * i + 1], ks, ks, -m.x, -m.y);
          fma2(x[4 * i + 2], x[4 * i + 3], ks, ks, -m.z, -m.w);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = ex2(x[i]);
        if (full) {
          float t0 = 0.f, t1 = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 v = ci[8 * q + i];
            fma2(x[4 * i], x[4 * i + 1], v.x, v.y, sum0, sum1);
            fma2(x[4 * i + 2], x[4 * i + 3], v.z, v.w, t0, t1);
            sum0 = x[4 * i], sum1 = x[4 * i + 1], t0 = x[4 * i + 2], t1 = x[4 * i + 3];
          }
          add2(sum0, sum1, t0, t1);
        } else {  // a row that does not see the position may have any sum
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int4 lim = cl[8 * q + i];
            const float4 v = ci[8 * q + i];
            sum0 += key < lim.x ? x[4 * i] * v.x : 0.f;
            sum1 += key < lim.y ? x[4 * i + 1] * v.y : 0.f;
            sum0 += key < lim.z ? x[4 * i + 2] * v.z : 0.f;
            sum1 += key < lim.w ? x[4 * i + 3] * v.w : 0.f;
          }
        }
      }
      tc_fence_before();
      warp_arrive(s_empty(b));
      if (lane == 0) mbar_arrive(q_empty(qb));
    }
  } else if (warp < 12) {
    const int r = tid - 256;
    const uint16_t* const q0 = (const uint16_t*)a.q;
    constexpr int kLag = L::COUNT - 2;  // tiles whose copies are still under way when the next are begun
    for (int g = 0; g < tiles + kLag; ++g) {
      const int b = g % L::COUNT, row = (rt0 + rank + 2 * g) * kM + r, tok = row / a.rep;
      if (g < tiles) {
        const int limit = row < p.rows && tok < sp.fresh ? sp.limit(a, tok) : 0;
        const float2 st = limit > 0 ? __ldg(p.stats + (size_t)zh * p.rows + row) : make_float2(0.f, 0.f);
        if (!wait(q_empty(b), (g / L::COUNT & 1) ^ 1)) goto out;
        copy_query<D>(base + L::Q + b * L::TILE, r,
                      limit > 0 ? q0 + (z * a.qs[0] + (h * a.rep + row % a.rep) * a.qs[1] + tok * a.qs[2]) : nullptr, q0, p.vec_q);
        col[b * 384 + r] = st.x == -INFINITY ? 0.f : st.x;
        col[b * 384 + 128 + r] = st.y;
        reinterpret_cast<int*>(col)[b * 384 + 256 + r] = limit;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (g >= kLag && tiles) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
        fence_proxy_async_smem();
        warp_arrive(q_full((g - kLag) % L::COUNT));
      }
    }
  } else {
    constexpr uint32_t IS = idesc_f16(kM, !FP16, false);
    const uint32_t kw = k_word(base + L::K), qw = k_word(base + L::Q);
    if (!wait(k_full, 0)) goto out;
    for (int g = 0; g < tiles; ++g) {
      const int b = g & 1, qs = g % L::COUNT;
      if (!wait(q_full(qs), g / L::COUNT & 1) || !wait(s_empty(b), (g >> 1 & 1) ^ 1)) goto out;
      tc_fence_after();
      const uint32_t kb = uniform(kw), qb = uniform(qw + qs * (L::TILE / 16)), to = uniform(tmem + b * 128);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) mma_ss(to, k_desc(kb, s), k_desc(qb, s), IS, s > 0, lane == 0);
      if (lane == 0) {
        tc_commit(s_full(b));
        tc_commit(q_empty(qs));
      }
      __syncwarp();
    }
  }
out:
  __syncwarp();
  if (warp == 12) {
    if (lane == 0) tc_commit(done);
    __syncwarp();
    mbar_wait(done, 0);
  }
  if (warp >= 4 && warp < 8) other[tid - 128] = sum0 + sum1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 256);
  const float sum = (sum0 + sum1) + (tid < kKeys ? other[tid] : 0.f);
  if (rank == 1 && tid < kKeys) other[tid] = sum;  // each thread's own word
  cluster_sync();
  if (rank == 0 && tid < kKeys && key < sp.len)
    c.weight[head + key] = a.weights_in[head + key] + (sum + __uint_as_float(peer_word(reinterpret_cast<const uint32_t*>(other) + tid, 1)));
  cluster_sync();  // the second CTA's shared memory stays until it was read
}

// ------------------------------------------------------------------ host
static PromptArgs plan_prompt(const AttendArgs& a, bool weights, int sms, size_t* bytes) {
  PromptArgs p;
  p.a = a;
  p.rows = a.N * a.rep;
  p.row_tiles = (p.rows + kRows - 1) / kRows;
  p.grid = sms;
  const size_t parts = (size_t)2 * sms * kRows * (a.c.D + 2) * 4;
  const size_t stats = weights ? (size_t)a.c.Z * a.c.H * p.rows * 8 : 0;
  p.parts = nullptr;
  p.stats = (float2*)parts;  // offset, for now
  *bytes = parts + stats;
  return p;
}

constexpr int kSms = 148;

size_t prompt_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  AttendArgs a;
  a.c = view(c), a.rep = Hq / c->H, a.N = N;
  size_t n;
  plan_prompt(a, weights, kSms, &n);
  return n;
}

template <void (*kernel)(PromptArgs)>
static int allow_smem(uint32_t bytes, int dev) {
  static std::atomic<bool> done[kDevices];  // per kernel and device
  if (done[dev].load(std::memory_order_relaxed)) return QFLASH_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
    return set_err(QFLASH_ERR_LAUNCH, "kv4 prompt: shared memory: %s", cudaGetErrorString(cudaGetLastError()));
  done[dev].store(true, std::memory_order_relaxed);
  return QFLASH_OK;
}

template <int D, bool FP16>
static int launch_prompt(const PromptArgs& p, int dev, cudaStream_t s) {
  if (int rc = allow_smem<prompt_kernel<D, FP16>>(Layout<D>::BYTES, dev)) return rc;
  prompt_kernel<D, FP16><<<p.grid, kPrompt, Layout<D>::BYTES, s>>>(p);
  if (int rc = check_launch("kv4 prompt", p.grid)) return rc;
  const unsigned n = 8 * p.grid + p.a.c.Z * p.row_tiles;
  launch_behind(prompt_finish_kernel<D, FP16>, n, 256, s, p);
  if (int rc = check_launch("kv4 prompt finish", n)) return rc;
  if (!p.stats) return QFLASH_OK;
  if (int rc = allow_smem<prompt_weights_kernel<D, FP16>>(WLayout<D>::BYTES, dev)) return rc;
  const unsigned nw = 2u * (unsigned)(p.a.c.Z * p.a.c.H) * ((p.a.c.C + kKeys - 1) / kKeys);
  prompt_weights_kernel<D, FP16><<<nw, kWeigh, WLayout<D>::BYTES, s>>>(p);
  return check_launch("kv4 prompt weights", nw);
}

int attend_prompt(const AttendArgs& a, bool fp16, void* ws, int dev, cudaStream_t s) {
  size_t n;
  PromptArgs p = plan_prompt(a, a.weights_in != nullptr, std::min(kSms, sm_count(dev)), &n);
  p.parts = (float*)ws;
  p.magic_k = fp16 ? kMagicFp16 : kMagicBf16, p.magic_v = kMagicBf16;
  p.stats = a.weights_in ? (float2*)((uint8_t*)ws + (size_t)p.stats) : nullptr;
  auto aligned = [](const void* q, const int64_t* st) { return (((uintptr_t)q | (st[0] * 2) | (st[1] * 2) | (st[2] * 2)) & 15) == 0; };
  p.vec_q = aligned(a.q, a.qs), p.vec_o = aligned(a.out, a.os);
  if (a.c.D == 64) return fp16 ? launch_prompt<64, true>(p, dev, s) : launch_prompt<64, false>(p, dev, s);
  return fp16 ? launch_prompt<128, true>(p, dev, s) : launch_prompt<128, false>(p, dev, s);
}

}  // namespace kv4
}  // namespace qfb
