// Pieces shared by the 8-bit KV cache kernels: the paged layout, the sequences of a call, and the
// int8 -> f16 conversion that feeds the tensor cores.
//
// The cache holds int8 codes [num_blocks, kv_heads, block_size, head_dim] for K and for V and one
// float32 scale per (block, kv head) of each; value = code * scale.  Token p of sequence b is slot
// p % block_size of block block_table[b, p / block_size].  A (block, kv head) tile is contiguous.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "internal.h"
#include "ptx.cuh"

namespace qhtp {
namespace kv8 {

// Scales below this count as zero when a block is written.  The attention kernels divide by V scales
// (see kv8_decode.cu): from 2^-64 up, 1 / scale summed over 2^31 keys stays far inside float32.
constexpr float kScaleMin = 5.421010862427522e-20f;  // 2^-64

struct Pages {
  int8_t* k;
  int8_t* v;
  float* k_scale;
  float* v_scale;
  long long num_blocks;
  int heads;      // kv heads
  int bs_log2;    // block_size = 1 << bs_log2
};

struct Seqs {
  const int32_t* table;   // [batch, max_blocks]
  long long table_stride;
  int max_blocks;
  int batch;
  const int32_t* start;   // [batch + 1] rows of each sequence, or null: `tokens` rows each
  int tokens;             // rows of each sequence, or (start given) the most of any
  long long total;        // rows in all (start given)
};

struct Rows {
  void* data;
  long long batch_stride, token_stride, head_stride;  // in elements; head_dim is contiguous
};

// Rows of sequence b: their number, and the index that token_stride multiplies for the first.  A start
// that lies outside [0, total] gives no rows.
__device__ __forceinline__ int seq_rows(const Seqs& s, int b, long long& first) {
  if (s.start == nullptr) {
    first = 0;
    return s.tokens;
  }
  const long long a = s.start[b], e = s.start[b + 1];
  first = a;
  return a < 0 || e > s.total || e <= a ? 0 : static_cast<int>(e - a);
}

// Block of a sequence's block index, or -1 where the table has none or names one outside the cache.
__device__ __forceinline__ long long block_of(const Seqs& s, const Pages& p, int b, long long idx) {
  if (idx < 0 || idx >= s.max_blocks) return -1;
  const long long id = s.table[b * s.table_stride + idx];
  return id >= 0 && id < p.num_blocks ? id : -1;
}

// Four int8 codes (one word) -> two half2, exactly: code + 128 is put into the low mantissa bits of
// the half 1024, and 1024 + 128 is taken off.  Three integer / half2 instructions per two codes less
// a shared xor, against four conversions.
__device__ __forceinline__ uint32_t sub_1152(uint32_t h) {
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  lo = sub_1152(prmt(w, 0x64646464u, 0x4140u));
  hi = sub_1152(prmt(w, 0x64646464u, 0x4342u));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float nan_f32() { return __uint_as_float(0x7fffffffu); }

// 16 bytes of T -> float32
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int n = 4;
  __device__ static void load(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  __device__ static uint4 store(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Vec<__half> {
  static constexpr int n = 8;
  __device__ static void load(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  __device__ static uint4 store(const float (&f)[8]) {
    return make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static void load(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static uint4 store(const float (&f)[8]) {
    return make_uint4(pack(f[0], f[1]), pack(f[2], f[3]), pack(f[4], f[5]), pack(f[6], f[7]));
  }
};

}  // namespace kv8

// kv8_cache.cu
struct Kv8Move {
  kv8::Pages pages;
  kv8::Seqs seqs;
  const int32_t* first;   // cache position of each sequence's first row
  kv8::Rows k, v;
  uint32_t dtype;
  int head_dim;
  cudaStream_t stream;
};
cudaError_t launch_kv8_write(const Kv8Move& m);
cudaError_t launch_kv8_read(const Kv8Move& m);

// Attention over the cache.  Query row r of a (sequence, kv head) is token r / group, head r % group of
// the kv head's group; token t of T stands at position length - T + t.
struct Kv8Attn {
  kv8::Pages pages;
  kv8::Seqs seqs;
  const int32_t* lengths;
  kv8::Rows q, out;
  float* lse;             // [rows, q_heads] or null
  int bf16;               // q and out: bf16, else f16
  int head_dim, q_heads, group;
  int causal, window;     // window 0: none
  float scale_log2;       // softmax scale * log2(e)
  int max_len;            // the caller's bound on the lengths (sizes the grid only)
  int prompt;             // kv8_prompt.cu, else kv8_decode.cu
  // A launch's plan: rows per CTA, row groups of a sequence (the most of any), and how the keys are cut.  fit > 0: into
  // chunks that the kernel sizes by the lengths, so that they are at most `fit` CTAs, of `chunk` keys at the least
  // (fit_place); fit = 0: into `chunks` of `chunk` keys, on a grid sized by max_len.
  int tile_rows, row_groups, chunk, chunks, fit;
  // Row groups of all sequences (of one kv head) that parts have room for.  packed: sequence b's are behind those that the
  // rows before it can fill (groups_before), else each sequence has room for row_groups.
  long long part_groups;
  int packed, tile_log2;  // tile_rows = 1 << tile_log2
  float* part;            // workspace: unnormalised rows, then their maxima and sums, then (fit) the sequences' cuts
  cudaStream_t stream;
};

namespace kv8 {

// Keys that rows [r0, r1) of a sequence of T tokens see, over all of the rows.
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span row_span(const Kv8Attn& a, int len, int T, int r0, int r1) {
  Span s{0, len};
  if (a.causal) s.hi = min(len, len - T + (r1 - 1) / a.group + 1);
  if (a.window) s.lo = max(0, len - T + r0 / a.group - a.window + 1);
  return s;
}
__device__ __forceinline__ int seq_length(const Kv8Attn& a, int b) {
  const long long cap = static_cast<long long>(a.seqs.max_blocks) << a.pages.bs_log2;
  const int len = max(a.lengths[b], 0);
  return len < cap ? len : static_cast<int>(cap);
}
// What a CTA works on: chunk `chunk` of `chunks`, `keys` long, of a (sequence, kv head, row group); `part`: its first row
// in the parts.
struct Place {
  int b, h, rg, chunk, chunks, keys;
  long long part;
};
// Chunk of a span: chunks start at a multiple of 32 keys, and the last takes what is left.
__device__ __forceinline__ Span chunk_span(const Place& p, const Span& s) {
  const long long lo = (s.lo & ~31) + static_cast<long long>(p.chunk) * p.keys;
  const long long hi = p.chunk == p.chunks - 1 ? s.hi : min(static_cast<long long>(s.hi), lo + p.keys);
  return lo < hi ? Span{static_cast<int>(lo), static_cast<int>(hi)} : Span{0, 0};
}
// Where the sequences' parts lie.  Of packed rows, sequence b's first row is row0 of all: the ones before it fill at most
// floor(row0 group / tile_rows) row groups and begin at most b more, one for each sequence.
__host__ __device__ __forceinline__ long long groups_before(const Kv8Attn& a, long long b, long long row0) {
  return a.packed ? ((row0 * a.group) >> a.tile_log2) + b : b * a.row_groups;
}
__host__ inline void place_parts(Kv8Attn& a) {
  const long long all = static_cast<long long>(a.seqs.batch) * a.row_groups;
  a.tile_log2 = 0;
  while ((1 << a.tile_log2) < a.tile_rows) ++a.tile_log2;
  a.packed = 1;
  a.part_groups = groups_before(a, a.seqs.batch, a.seqs.total);
  if (a.seqs.start == nullptr || a.part_groups >= all) a.packed = 0, a.part_groups = all;
}
// Offset of a (sequence, kv head, row group, chunk) part in rows.
__device__ __forceinline__ long long part_row(const Kv8Attn& a, int b, long long row0, int h, int rg, int c) {
  return (((groups_before(a, b, row0) + rg) * a.pages.heads + h) * a.chunks + c) * a.tile_rows;
}
__host__ __device__ __forceinline__ long long part_rows(const Kv8Attn& a) {
  return (a.fit ? a.fit : a.part_groups * a.pages.heads * a.chunks) * a.tile_rows;
}

// Cutting the keys by the lengths.  A grid sized on the host has to be sized for the longest sequence that there may be:
// lengths that differ, or a loose max_len, then leave it half empty.  Here every CTA looks at all lengths and finds the
// smallest chunk (a multiple of 128 keys, a.chunk at the least) whose chunks are at most a.fit, and then which one is
// its own: the chunks of a sequence follow one another, heads fastest.  It costs a CTA some 3 us of its start (measured figures
// are at the plans).  The cut, and with it a sequence's roundings, depends on all lengths of the call; the same lengths give
// the same bits.
constexpr int kFitBatch = 512;  // sequences of a call with fit, at most
// A sequence's cut, for the kernel that joins the chunks: its first CTA, its chunks (of each row group), their length,
// and its row groups.
__device__ __forceinline__ int4* cuts_of(const Kv8Attn& a) {
  return reinterpret_cast<int4*>(a.part + part_rows(a) * (a.head_dim + 2));
}
// A quotient that rounding leaves one too high or too low does no harm: the last chunk takes what is left, and an empty
// one ends at once.
__device__ __forceinline__ int chunks_of(int span, float per_key) { return max(__float2int_ru(span * per_key), 1); }
// The same value of every thread as one that the compiler knows to be: it stays in a uniform register.
__device__ __forceinline__ int uniform(int x) { return static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(x))); }
// The CTA's place; false: none is left for it.  memory: room for a.seqs.batch entries, used until this returns (and, by
// the async proxy's clock, done with).  Every thread of the block takes part, warps beside one another do the same.
__device__ __forceinline__ bool fit_place(const Kv8Attn& a, int cta, int2* memory, Place& p) {
  const int lane = threadIdx.x & 31, n = a.seqs.batch;
  // the keys that a row group of a sequence sees at the most, from a multiple of 32 on, and its CTAs of a chunk
  auto look = [&](int b) {
    long long row0;
    const long long R = static_cast<long long>(seq_rows(a.seqs, b, row0)) * a.group;
    const int groups = static_cast<int>(min(static_cast<long long>(a.row_groups), (R + a.tile_rows - 1) / a.tile_rows));
    int span = seq_length(a, b);
    if (a.window) span = min(span, min(a.window, 1 << 29) + a.tile_rows / a.group + 32);
    return make_int2(span + 31, groups * a.pages.heads);
  };
  // the first 32 sequences are in registers, the others, where there are more, in memory
  const int2 own = lane < n ? look(lane) : make_int2(0, 0);
  if (n > 32) {
#pragma unroll 1
    for (int b = 32 + threadIdx.x; b < n; b += blockDim.x) memory[b] = look(b);
    __syncthreads();
  }
  auto seq = [&](int b) { return b < 32 ? own : memory[b]; };  // b % 32 == lane
  long long total = 0;
  int longest = 0, items = 0;
#pragma unroll 1
  for (int b = lane; b < n; b += 32) {
    const int2 s = seq(b);
    total += static_cast<long long>(s.x) * s.y;
    longest = max(longest, s.x), items += s.y;
  }
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  longest = uniform(longest);
  items = __reduce_add_sync(0xffffffffu, items);
  auto fits = [&](int tiles) {
    const float per_key = __fdividef(1.0f, tiles * 128);
    int sum = 0;
#pragma unroll 1
    for (int b = lane; b < n; b += 32) sum += chunks_of(seq(b).x, per_key) * seq(b).y;
    return __reduce_add_sync(0xffffffffu, sum) <= a.fit;
  };
  // Chunks of total / fit keys are too many, except where nothing is left over.  Those of total / (fit - items) should be
  // few enough, since an item has at most one chunk that is not full; those of the longest sequence are, as there are no
  // more than fit items.
  auto share = [&](int ctas) {
    return __float2int_rd(fminf(__fdividef(static_cast<float>(total), static_cast<float>(ctas)), 1e9f));
  };
  const int most = max(longest, a.chunk) / 128 + 1;
  int lo = min(max(a.chunk, share(a.fit)) / 128, most);
  int hi = items < a.fit ? max(min(share(a.fit - items) / 128 + 1, most), lo) : most;
  int mid = hi;
#pragma unroll 1
  do {
    if (fits(mid))
      hi = mid;
    else if (mid == hi)
      lo = hi + 1, hi = most;  // the guess was too low
    else
      lo = mid + 1;
    mid = (lo + hi) >> 1;
  } while (lo < hi);
  p.keys = uniform(hi * 128);
  const float per_key = __fdividef(1.0f, p.keys);
  bool there = false;
  int before = 0;  // CTAs of the sequences so far
#pragma unroll 1
  for (int b0 = 0; b0 < n && !there; b0 += 32) {
    const int2 s = b0 + lane < n ? seq(b0 + lane) : make_int2(0, 0);
    const int mine = chunks_of(s.x, per_key) * s.y;
    int upto = mine;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    upto += before;
    const unsigned found = __ballot_sync(0xffffffffu, cta < upto);
    if (found) {
      const int at = __ffs(found) - 1;
      const int first = uniform(__shfl_sync(0xffffffffu, upto - mine, at)), one = uniform(__shfl_sync(0xffffffffu, s.y, at));
      p.b = uniform(b0 + at);
      p.chunk = uniform((cta - first) / one);
      const int item = cta - first - p.chunk * one, rg = uniform(item / a.pages.heads);
      p.h = item - rg * a.pages.heads;
      p.rg = one / a.pages.heads - 1 - rg;  // the longest (the last of a causal sequence) first
      p.chunks = uniform(chunks_of(__shfl_sync(0xffffffffu, s.x, at), per_key));
      p.part = static_cast<long long>(cta) * a.tile_rows;
      if (cta == first && threadIdx.x == 0) cuts_of(a)[p.b] = make_int4(first, p.chunks, p.keys, one);
      there = true;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  if (n > 32) {
    fence_proxy_async_smem();
    __syncthreads();
  }
  return there;
}

// Exponents are taken to m - kLift, so that a row's p are 2^7 where t = m.  As f16 operands they keep 11 bits down to 2^-14,
// 2^-21 of that, and below it are off by 2^-25, 2^-32 of it: 2^20 keys of small p, which may be all of the output where the
// largest p's key has a small value, then lose no more than f16's 11 bits do.  (At kLift 0 thousands of keys of 2^-25 each were
// off by a quarter.)  The prompt kernels let p pass that by 2^8 (kGrow): 2^15, inside f16.
constexpr float kLift = 7.0f;

// mbar_wait for a whole warp: every lane goes on, or none does.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

// A block's constants for the softmax: with c = scale * log2(e) * k_scale and w = v_scale, a key's
// exponent is q . code * c + log2(w), and 1 / w takes w out of the row's sum again.  A v_scale below
// kScaleMin counts as zero: w is kScaleMin then, and inv_w = kZeroTile tells that the codes add nothing.
struct BlockScales {
  float c, log2_w, inv_w;
};
constexpr float kZeroTile = 36893488147419103232.0f;  // 2^65
struct RawScales {
  float k, v;
};
__device__ __forceinline__ RawScales raw_scales(const Kv8Attn& a, long long id, int h) {
  if (id < 0) return {nan_f32(), nan_f32()};
  const long long t = id * a.pages.heads + h;
  return {a.pages.k_scale[t], a.pages.v_scale[t]};
}
__device__ __forceinline__ BlockScales fold_scales(const Kv8Attn& a, const RawScales& s) {
  const float v = s.v < kScaleMin ? kScaleMin : s.v;  // a NaN stays
  return {s.k * a.scale_log2, log2f(v), s.v < kScaleMin ? kZeroTile : 1.0f / v};
}

// 2^-e and the factor 2^e that brings a row of largest magnitude `top` to [2^14, 2^15): q then fits f16 without
// overflow, and every element within 2^-29 of the largest keeps all of its bits.
__device__ __forceinline__ void row_factor(float top, float& up, float& down) {
  const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;  // top >= 0
  if (top == 0.0f || e >= 128) {  // nothing to scale, or not finite
    up = down = 1.0f;
    return;
  }
  // e >= -126 (a subnormal counts as 2^-127): 14 - e <= 141 can pass 2^127, so it is capped there
  const int up_e = min(14 - max(e, -127), 126);
  up = __uint_as_float(static_cast<uint32_t>(up_e + 127) << 23);
  down = __uint_as_float(static_cast<uint32_t>(127 - up_e) << 23);
}

// Eight elements of a finished row: out = o / sum, and (with the row's first eight) its lse.  A row that
// sees no key has sum 0: zeros, and an lse of -infinity.
__device__ __forceinline__ void write_row8(const Kv8Attn& a, int b, long long row0, int row, int h, int d0,
                                           const float (&o)[8], float sum, float top) {
  const int t = row / a.group, head = h * a.group + row - t * a.group;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = o[e] * inv;
  uint16_t* to = static_cast<uint16_t*>(a.out.data) + b * a.out.batch_stride + (row0 + t) * a.out.token_stride +
                 head * a.out.head_stride + d0;
  *reinterpret_cast<uint4*>(to) = a.bf16 ? Vec<__nv_bfloat16>::store(v) : Vec<__half>::store(v);
  if (a.lse != nullptr && d0 == 0) {
    const long long at = (a.seqs.start ? row0 : static_cast<long long>(b) * a.seqs.tokens) + t;
    a.lse[at * a.q_heads + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945309f;
  }
}

}  // namespace kv8

// kv8_decode.cu: rows in groups of 8 to 32 on warp-level MMAs, for few rows per (sequence, kv head)
void kv8_decode_plan(Kv8Attn& a, int sms);
cudaError_t launch_kv8_decode(const Kv8Attn& a);
// kv8_prompt.cu: rows in tiles of 128 or 256 on tcgen05
void kv8_prompt_plan(Kv8Attn& a, int sms);
cudaError_t launch_kv8_prompt(const Kv8Attn& a);
// kv8_prompt2.cu: tiles of 256 rows, head_dim 64 and 128
cudaError_t launch_kv8_prompt2(const Kv8Attn& a);

// joins the chunks of a launch
cudaError_t launch_kv8_combine(const Kv8Attn& a);
// the current device's error words of the attention kernels: a wait that gave up leaves its code there
cudaError_t kv8_decode_word(int** word);
cudaError_t kv8_prompt_word(int** word);
cudaError_t kv8_prompt2_word(int** word);
// reads and clears one; synchronizes
inline cudaError_t kv8_take_error(int* word, int* code, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyAsync(code, word, sizeof(int), cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, sizeof(int), stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  return e;
}
// Runs `set` once per device (again where it failed).
template <typename F>
inline cudaError_t once_per_device(std::atomic<bool> (&done)[64], F set) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t r = set();
  if (r == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
  return r;
}
inline size_t kv8_part_bytes(const Kv8Attn& a) {
  if (a.chunks <= 1 && a.fit == 0) return 0;
  return static_cast<size_t>(kv8::part_rows(a)) * (a.head_dim + 2) * sizeof(float) + (a.fit ? a.seqs.batch * sizeof(int4) : 0);
}

}  // namespace qhtp
