// Attention of many query rows (prompts, pieces of prompts) over the 8-bit paged KV cache, on tcgen05.
//
// The mathematics is kv8_decode.cu's: exponents t = q . ck * (scale log2(e) sk) + log2(sv), outputs
// sum 2^(t - m) cv / sum 2^(t - m) / sv, the int8 codes as f16 operands, V's scale in the exponent.
//
// A CTA owns SLOTS tiles of 128 query rows (the tokens and heads of one kv head's group, packed) and walks
// over the keys 64 at a time:
//   K and V converters (a warpgroup each) bring codes from the paged cache by bulk copies into a staging tile (a 16-key
//     group of a head is contiguous in its block) and write them as f16 into 128-byte-swizzled images
//     [key][64 head_dim], three or four units ahead: K-major for Q K^T, and the same bytes MN-major for P V;
//   one warp issues the MMAs: S = Q K^T into tensor memory, O += P V with P read from tensor memory;
//   a softmax warpgroup per slot, a thread per row: S from tensor memory, P back over it as f16.
// Each slot has two S buffers, so that the softmax of one unit runs under the MMAs of its neighbours and of the other
// slot.  Q stands in tensor memory where that has room beside S and O (all but two slots of head_dim 128): an MMA then
// reads 2 KB of shared memory where it reads 6, and those are what its rate hangs on at 64 keys.
//
// m is raised, and O rescaled, only when a row's maximum has grown by more than 2^8: p then stays below
// 2^8, far inside f16, and most tiles leave O alone.
#include <algorithm>

#include "kv8.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kKeys = 64;              // keys of a unit
constexpr int kPanel = kKeys * 128;    // bytes of a [64 keys][64 f16] swizzled image
constexpr int kQPanel = 128 * 128;     // and of a [128 rows][64 f16] one
// pairs of a 16-key group whose exponentials are computed by polynomial, a bit each
constexpr uint32_t kPoly = 0x00;
constexpr float kGrow = 8.0f;          // log2 of how far p may pass 1 before m follows

template <int D, int SLOTS>
struct Shape {
  static constexpr int panels = D / 64;
  static constexpr int unit = panels * kPanel;                  // 64 keys of K or V
  static constexpr int units = D == 256 ? 3 : 4;                // of K, and of V
  static constexpr int q_tile = panels * kQPanel;
  // Q's image: where tensor memory takes Q and there is no room for both, it passes through V's last units
  static constexpr int q_smem = D == 256 ? 0 : SLOTS * q_tile;
  static constexpr int staging = 2 * kKeys * D;                 // codes on their way
  static constexpr int smem = q_smem + 2 * units * unit + staging + 1024;
  static_assert(smem + 2048 <= 227 * 1024, "shared memory");
  static constexpr int threads = (SLOTS + 3) * 128;
  // registers of a thread: at launch (the most that the threads leave room for), and by role; the roles' sum is the launch's
  static constexpr int regs = SLOTS == 2 ? 96 : 128;
  static constexpr int softmax_regs = SLOTS == 2 ? 144 : 184;
  static constexpr int convert_regs = SLOTS == 2 ? 72 : 120;
  static constexpr int mma_regs = SLOTS == 2 ? 48 : 80;
  static_assert(convert_regs <= regs && SLOTS * softmax_regs + 2 * convert_regs + mma_regs <= (SLOTS + 3) * regs, "registers");
  // tensor memory columns: S buffers from 0 (64 each, two per slot), O, Q
  static constexpr bool q_tmem = SLOTS == 1 || D == 64;
  static constexpr int q_col = SLOTS == 1 ? 128 : 384;
  static constexpr int o_col = 256;
  static_assert(o_col + SLOTS * D <= 512 && (!q_tmem || (SLOTS == 1 ? q_col + D / 2 <= o_col : o_col + SLOTS * D <= q_col)),
                "tensor memory");
};

struct Barriers {
  uint64_t q_full[2], k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[4], p_full[4], pv_done[2], drained, staged[2];
};

template <int N>
__device__ __forceinline__ void reg_alloc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_free() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// (a.x * b + c, a.y * b + c) in one instruction
__device__ __forceinline__ float2 fma2(float x, float y, float b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 u, v, w, z;\n\t"
      "mov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %4};\n\tmov.b64 w, {%5, %5};\n\t"
      "fma.rn.f32x2 z, u, v, w;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x), "f"(y), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 u, v, z;\n\t"
      "mov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\t"
      "add.rn.f32x2 z, u, v;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 u, v, w, z;\n\t"
      "mov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmov.b64 w, {%6, %6};\n\t"
      "fma.rn.f32x2 z, u, v, w;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c));
  return r;
}
// 2^t of a pair on the FMA pipe: t = n + f with n the nearest integer (it is left in the low bits of t + 1.5 2^23)
// and |f| <= 1/2, 2^f by the degree-4 polynomial of least relative error there (2.6e-6, found by Remez exchange), n added
// to the exponent.  t below -126 counts as -126.
__device__ __forceinline__ float2 ex2_poly(float2 t) {
  t.x = fmaxf(t.x, -126.0f), t.y = fmaxf(t.y, -126.0f);
  const float2 big = add2(t, make_float2(12582912.0f, 12582912.0f));
  const float2 n = add2(big, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = add2(t, make_float2(-n.x, -n.y));
  float2 p = fma2(f.x, f.y, 0.009570102207362652f, 0.05591785907745361f);
  p = fma2(p, f, 0.240247443318367f);
  p = fma2(p, f, 0.6931217908859253f);
  p = fma2(p, f, 0.9999992847442627f);
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(big.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(big.y) << 23)));
}
// Keeps uses of what tcgen05.ld wrote behind the wait for it: the wait itself does not name the registers.
template <int N>
__device__ __forceinline__ void pin(uint32_t (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(x[i]));
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// Low word of a descriptor of a 128-byte-swizzled image: start address and, for MN-major operands, the distance of
// 64-element groups; the high word (1024 bytes between 8-row atoms, version 1, swizzle) is kDescHi.  Steps are added to
// the low word in units of 16 bytes.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t at, uint32_t lbo) { return (at >> 4) | ((lbo >> 4) << 16); }
// The MMAs and commits are predicated on `leader`, not branched around: the code stays converged, and the compiler keeps
// addresses and descriptors in uniform registers.
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// A in tensor memory: one 32-bit column holds two consecutive K elements
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void arrive(uint32_t leader, uint32_t bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
               "r"(leader)
               : "memory");
}
// 16-byte chunk c of row r in a swizzled image
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
  return static_cast<uint32_t>(r * 128 + (((c ^ r) & 7) << 4));
}

// The rows of one slot as f16 into its image, rows of bf16 scaled by a power of two each.  D / 8 lanes a row, all of a
// warp's rows in flight at once.
template <int D>
__device__ __forceinline__ void load_q(const Kv8Attn& a, int b, int h, long long row0, int r0, int r1, uint8_t* img,
                                       float* down_at, int warp, int lane) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // rows of a load
  constexpr int kBatch = D == 256 ? 16 : 32 / kRows;  // loads in flight
  const int sub = lane / kLanes, c = lane % kLanes;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q.data) + b * a.q.batch_stride + row0 * a.q.token_stride +
                            static_cast<long long>(h) * a.group * a.q.head_stride + 8 * c;
  // token and head of the lane's next row
  int row = r0 + warp * 32 + sub;
  int t = row / a.group, head = row - t * a.group;
#pragma unroll 1
  for (int base = 0; base < 32 / kRows; base += kBatch) {
    uint4 w[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (row < r1) w[i] = __ldg(reinterpret_cast<const uint4*>(q + t * a.q.token_stride + head * a.q.head_stride));
      row += kRows;
      head += kRows;
      while (head >= a.group) head -= a.group, ++t;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = warp * 32 + (base + i) * kRows + sub;
      float down = 1.0f;
      if (a.bf16) {
        float x[8];
        Vec<__nv_bfloat16>::load(w[i], x);
        // bf16 magnitudes are ordered like their bits: the largest of the lane's, then of the row's
        uint32_t top = __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu),
                                __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = max(top & 0xffffu, top >> 16);
        float up;
        row_factor(__uint_as_float(top << 16), up, down);
        w[i] = make_uint4(pack_half2(x[0] * up, x[1] * up), pack_half2(x[2] * up, x[3] * up),
                          pack_half2(x[4] * up, x[5] * up), pack_half2(x[6] * up, x[7] * up));
      }
      *reinterpret_cast<uint4*>(img + (c >> 3) * kQPanel + swizzled(r, c & 7)) = w[i];
      if (c == 0) down_at[r] = down;
    }
  }
}

// The word that a wait of a kernel here, having given up, leaves its code in.
__device__ int g_error;

// A row's view of a unit: the group constants, and the columns that the row sees.  CAREFUL below: the unit has columns
// that not every row sees, or a group whose scales are not plain.
struct View {
  const float4* scale;
  float down;
  int lo, hi;
};

// The largest exponent of the row in this unit, or `top` where that is larger.
template <bool CAREFUL>
__device__ __forceinline__ float row_max(const View& k, const uint32_t (&x)[2][32], float top) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float4 sc = k.scale[c];
    const uint32_t* const v = &x[c >> 1][16 * (c & 1)];
    if constexpr (CAREFUL) {
      float best = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = 16 * c + e;
        best = fmaxf(best, col < k.hi && col >= k.lo ? __uint_as_float(v[e]) : -INFINITY);
      }
      if (best != -INFINITY) top = fmaxf(top, fmaf(best, sc.x * k.down, sc.y));
    } else {
      float best[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
      for (int e = 2; e < 14; e += 4) {
        best[0] = max3(best[0], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
        best[1] = max3(best[1], __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
      }
      best[0] = max3(best[0], __uint_as_float(v[14]), __uint_as_float(v[15]));
      top = fmaxf(top, fmaf(fmaxf(best[0], best[1]), sc.x * k.down, sc.y));
    }
  }
  return top;
}

// p as f16 pairs into w; returns l with the row's sum added.
template <bool CAREFUL>
__device__ __forceinline__ float row_exp(const View& k, const uint32_t (&x)[2][32], float base, float l, uint32_t (&w)[2][16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float4 sc = k.scale[c];
    const uint32_t* const v = &x[c >> 1][16 * (c & 1)];
    uint32_t* const to = &w[c >> 1][8 * (c & 1)];
    const float f = sc.x * k.down, off = sc.y - base;
    float2 sum[2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      float2 t = fma2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), f, off);
      if (!CAREFUL && kPoly >> (e / 2) & 1)
        t = ex2_poly(t);
      else
        t.x = ex2(t.x), t.y = ex2(t.y);
      if constexpr (CAREFUL) {
        const int col = 16 * c + e;
        t.x = col < k.hi && col >= k.lo ? t.x : 0.0f;
        t.y = col + 1 < k.hi && col + 1 >= k.lo ? t.y : 0.0f;
      }
      sum[(e >> 1) & 1] = e < 4 ? t : add2(sum[(e >> 1) & 1], t);
      to[e / 2] = pack_half2(t.x, t.y);
    }
    sum[0] = add2(sum[0], sum[1]);
    const float add = sum[0].x + sum[0].y;
    if constexpr (CAREFUL) {
      const bool zero = sc.z == kZeroTile;  // a tile of V whose scale counts as zero
      if (add != 0.0f) l = fmaf(add, zero ? 0.5f * kZeroTile : sc.z, l);  // hidden keys add nothing, whatever their scale
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = zero ? 0u : to[e];
    } else {
      l = fmaf(add, sc.z, l);
    }
  }
  return l;
}

template <int D, int SLOTS>
__global__ void __launch_bounds__(Shape<D, SLOTS>::threads, 1) kv8_prompt_kernel(const Kv8Attn a) {
  using S = Shape<D, SLOTS>;
  int* const err = &g_error;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t s_tmem;
  __shared__ float s_down[SLOTS * 128];
  __shared__ float4 s_scale[8][4];       // (c, log2 w, 1 / w, care) of a unit's 16-key groups, eight units deep

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // heads fastest, the longest row groups (the last of a causal sequence) first
  const int h = blockIdx.x / a.chunks, chunk = blockIdx.x - h * a.chunks, b = blockIdx.y,
            rg = a.row_groups - 1 - blockIdx.z;
  long long row0;
  const int T = seq_rows(a.seqs, b, row0);
  const int R = T * a.group, r0 = rg * SLOTS * 128;
  if (r0 >= R) return;
  const int r1 = min(R, r0 + SLOTS * 128);
  const int len = seq_length(a, b);
  const Span all = row_span(a, len, T, r0, r1);
  const Span keys = chunk_span(a, all, chunk);
  const int units = keys.lo < keys.hi ? (keys.hi - keys.lo + kKeys - 1) / kKeys : 0;
  if (units == 0 && chunk > 0) return;

  uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* const k_img = smem + S::q_smem;
  uint8_t* const v_img = k_img + S::units * S::unit;
  uint8_t* const stage_img = v_img + S::units * S::unit;
  uint8_t* const q_img = S::q_smem ? smem : v_img + S::unit;
  static_assert(S::q_smem != 0 || S::q_tile <= (S::units - 1) * S::unit, "Q in V's units");

  constexpr int kConvK = SLOTS * 4, kConvV = kConvK + 4, kMma = kConvV + 4;  // first warps of the roles
  if (warp == kMma) {
    tmem_alloc(&s_tmem, 512);
    if (lane == 0) {
      for (int i = 0; i < 4; ++i) {
        mbar_init(&bar.k_full[i], 128);
        mbar_init(&bar.v_full[i], 128);
        mbar_init(&bar.k_empty[i], 1);
        mbar_init(&bar.v_empty[i], 1);
        mbar_init(&bar.s_full[i], 2);  // the MMAs, and the issuing thread's own arrival
        mbar_init(&bar.p_full[i], 128);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bar.q_full[i], 128);
        mbar_init(&bar.pv_done[i], 1);
        mbar_init(&bar.staged[i], 1);
      }
      mbar_init(&bar.drained, 1);
      fence_barrier_init();
    }
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < kConvK) {
    // ------------------------------------------------------------------------------- softmax, a thread per row
    reg_alloc<S::softmax_regs>();
    const int slot = warp >> 2, wq = warp & 3, r = r0 + slot * 128 + wq * 32 + lane;
    const int sr0 = r0 + slot * 128, sr1 = min(r1, sr0 + 128);  // the slot's rows (none: sr0 >= sr1)
    const uint32_t lanes = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const uint32_t o_at = lanes + S::o_col + slot * D;
    float m = -INFINITY, l = 0.0f;
    if (units > 0 && sr0 < sr1) {
      load_q<D>(a, b, h, row0, sr0, sr1, q_img + slot * S::q_tile, s_down + slot * 128, wq, lane);
      __syncwarp();
      const float down = s_down[slot * 128 + wq * 32 + lane];
      if constexpr (S::q_tmem) {
        const int qr = wq * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t x[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 4 * c + e;
            const uint4 v = *reinterpret_cast<const uint4*>(q_img + slot * S::q_tile + (at >> 3) * kQPanel + swizzled(qr, at & 7));
            x[4 * e] = v.x, x[4 * e + 1] = v.y, x[4 * e + 2] = v.z, x[4 * e + 3] = v.w;
          }
          tmem_st16(lanes + S::q_col + slot * (D / 2) + 16 * c, x);
        }
        tmem_st_wait();
        tc_fence_before();
      } else {
        fence_proxy_async_smem();
      }
      mbar_arrive(&bar.q_full[slot]);
      const int p = len - T + r / a.group;
      const int row_hi = r >= sr1 ? 0 : a.causal ? min(len, p + 1) : len, row_lo = a.window ? p - a.window + 1 : 0;
      // every row of the slot sees the keys [all_lo, all_hi)
      const int all_hi = a.causal ? len - T + sr0 / a.group + 1 : len;
      const int all_lo = a.window ? len - T + (sr1 - 1) / a.group - a.window + 1 : 0;
      for (int i = 0; i < units; ++i) {
        const int buf = slot * 2 + (i & 1);
        const uint32_t s_at = lanes + buf * 64;
        if (!warp_wait(&bar.s_full[buf], (i >> 1) & 1, err, kErrTimeoutAccum)) break;
        tc_fence_after();
        uint32_t x[2][32];
        tmem_ld32(s_at, x[0]);
        tmem_ld32(s_at + 32, x[1]);
        const int key0 = keys.lo + i * kKeys;
        const View k{s_scale[i & 7], down, row_lo - key0, row_hi - key0};
        const bool careful = key0 + kKeys > all_hi || key0 < all_lo || k.scale[0].w != 0.0f;
        tmem_ld_wait();
        pin(x[0]), pin(x[1]);
        const float top = careful ? row_max<true>(k, x, m) : row_max<false>(k, x, m);
        // raise m where it pays; rows of a warp move together
        if (__any_sync(0xffffffffu, top > m + kGrow || (m == -INFINITY && top != -INFINITY))) {
          const float alpha = m == -INFINITY ? 0.0f : ex2(m - top);
          if (i > 0) {
            if (!warp_wait(&bar.pv_done[slot], (i - 1) & 1, err, kErrTimeoutAccum)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_at + 16 * c, o);
              tmem_ld_wait();
              pin(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(o_at + 16 * c, o);
            }
          }
          l *= alpha;
          m = top;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        uint32_t w[2][16];
        l = careful ? row_exp<true>(k, x, base, l, w) : row_exp<false>(k, x, base, l, w);
        tmem_st16(s_at, w[0]);
        tmem_st16(s_at + 16, w[1]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar.p_full[buf]);
      }
      // the last product may be two phases ahead of what this warp has seen (S of a unit comes before P V of the one before
      // it), and a parity tells only one: both are waited for
      if (units > 1) warp_wait(&bar.pv_done[slot], (units - 2) & 1, err, kErrTimeoutAccum);
      warp_wait(&bar.pv_done[slot], (units - 1) & 1, err, kErrTimeoutAccum);
      tc_fence_after();
    }
    // the rows
    if (sr0 < sr1) {
      const float base = m == -INFINITY ? 0.0f : m;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const bool live = r < sr1;
      const int t = r / a.group, head = h * a.group + r - t * a.group;
      const long long part = part_row(a, b, h, rg, chunk) + slot * 128 + wq * 32 + lane;
      uint16_t* out = static_cast<uint16_t*>(a.out.data) + b * a.out.batch_stride + (row0 + t) * a.out.token_stride +
                      head * a.out.head_stride;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[32];
        if (units > 0) {
          tmem_ld32(o_at + 32 * c, x);
          tmem_ld_wait();
          pin(x);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0;
        }
        __syncwarp();
        if (live && a.chunks == 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x[e + i]) * inv;
            *reinterpret_cast<uint4*>(out + 32 * c + e) = a.bf16 ? Vec<__nv_bfloat16>::store(v) : Vec<__half>::store(v);
          }
        } else if (live) {
          uint4* to = reinterpret_cast<uint4*>(a.part + part * D + 32 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e) to[e] = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        }
        __syncwarp();
      }
      if (live && a.chunks == 1 && a.lse != nullptr) {
        const long long at = (a.seqs.start ? row0 : static_cast<long long>(b) * a.seqs.tokens) + t;
        a.lse[at * a.q_heads + head] = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.693147180559945309f;
      } else if (live && a.chunks > 1) {
        float* ml = a.part + part_rows(a) * D + 2 * part;
        ml[0] = base, ml[1] = l;
      }
    }
  } else if (warp < kMma) {
    // ------------------------------------------------------------------------------- codes to f16 images
    if constexpr (S::convert_regs < S::regs) reg_free<S::convert_regs>();
    constexpr int kStep = 128 / (D / 8), kSteps = kKeys / kStep;
    const bool is_v = warp >= kConvV;
    const int t = threadIdx.x - (is_v ? kConvV : kConvK) * 32;
    // A thread has chunk c (eight codes, 16 bytes as f16) of the rows row, row + kStep, ...: loads and stores of a
    // warp are whole rows, without bank conflicts.
    const int c = t % (D / 8), row = t / (D / 8);
    uint8_t* const stage = stage_img + (is_v ? kKeys * D : 0);
    const uint32_t from = smem_u32(stage) + row * D + c * 8;
    const uint32_t to = smem_u32(is_v ? v_img : k_img) + (c >> 3) * kPanel + swizzled(row, c & 7);
    const bool copies = (warp & 3) == 0, scales = warp == kConvK;
    const int bs_log2 = a.pages.bs_log2, bs = 1 << bs_log2;
    uint64_t* const staged = &bar.staged[is_v ? 1 : 0];
    uint64_t* const full = is_v ? bar.v_full : bar.k_full;
    uint64_t* const empty = is_v ? bar.v_empty : bar.k_empty;
    const int8_t* const codes = is_v ? a.pages.v : a.pages.k;
    // block of the unit's 16-key group `lane` (of four); -1: none
    auto ids_of = [&](int i) {
      const int key = keys.lo + i * kKeys + 16 * (lane & 3);
      return i < units && key < keys.hi ? static_cast<int>(block_of(a.seqs, a.pages, b, key >> bs_log2)) : -1;
    };
    int issued = 0;
    // groups that there are none of keep the codes that happen to be there: they are hidden, or their scales are NaN
    auto copy = [&](int i, int id) {
      ++issued;
      const bool there = lane < 4 && id >= 0;
      const int n = __popc(__ballot_sync(0xffffffffu, there));
      if (lane == 0) mbar_arrive_expect_tx(staged, n * 16 * D);
      __syncwarp();
      if (there) {
        const int slot = (keys.lo + i * kKeys + 16 * lane) & (bs - 1);
        bulk_load(stage + lane * 16 * D, codes + (((static_cast<long long>(id) * a.pages.heads + h) << bs_log2) + slot) * D,
                  16 * D, staged);
      }
    };
    int id = ids_of(0), id_next = ids_of(1);
    RawScales sc{}, sc_next{};
    if (units > 0) {
      if (copies) copy(0, id);
      if (scales) sc = raw_scales(a, id, h);
    }
    bool ok = true;
    for (int i = 0; i < units; ++i) {
      const int at = i % S::units;
      const int id_after = ids_of(i + 2);
      if (scales) sc_next = raw_scales(a, id_next, h);
      ok = warp_wait(staged, i & 1, err, kErrTimeoutFull);
      if (!ok) break;
      uint2 raw[kSteps];
#pragma unroll
      for (int e = 0; e < kSteps; ++e) raw[e] = lds64(from + e * kStep * D);
      named_barrier(is_v ? 2 : 1, 128);  // the staging tile is read
      if (copies && i + 1 < units) copy(i + 1, id_next);
      if (i >= S::units) ok = warp_wait(&empty[at], ((i / S::units) - 1) & 1, err, kErrTimeoutEmpty);
      if (S::q_smem == 0 && is_v && i == 1) ok = warp_wait(&bar.q_full[0], 0, err, kErrTimeoutEmpty);  // Q has passed
      if (!ok) break;
      if (scales) {
        // .w: a group whose scales need care (zero, or not finite)
        const BlockScales f = fold_scales(a, sc);
        const bool odd = !(f.inv_w < kZeroTile) || !isfinite(f.c);
        const float care = __any_sync(0xffffffffu, odd) ? 1.0f : 0.0f;
        if (lane < 4) s_scale[i & 7][lane] = make_float4(f.c, f.log2_w, f.inv_w, care);
      }
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        uint32_t u[4];
        codes_to_half2(raw[e].x, u[0], u[1]);
        codes_to_half2(raw[e].y, u[2], u[3]);
        // rows 4 apart (head_dim 256) differ in bit 2 of the swizzle, rows 8 apart not at all
        const uint32_t flip = kStep == 4 && (e & 1) ? 64u : 0u;
        sts128((to ^ flip) + at * S::unit + e * kStep * 128, u[0], u[1], u[2], u[3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(&full[at]);
      id = id_next, id_next = id_after, sc = sc_next;
    }
    // a wait gave up: copies under way end before the block does
    if (!ok && copies) warp_wait(staged, (issued - 1) & 1, err, kErrTimeoutOther);
  } else {
    // ------------------------------------------------------------------------------- the MMAs
    reg_free<S::mma_regs>();
    if (warp == kMma && units > 0) {
      const int slots = SLOTS == 2 && r0 + 128 < r1 ? 2 : 1;
      constexpr uint32_t id_qk = idesc_f16(128, kKeys), id_pv = idesc_f16(128, D, 1);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), leader = elect_one();
      const uint32_t q_desc = desc_lo(smem_u32(q_img), 16), k_desc = desc_lo(smem_u32(k_img), 16),
                     v_desc = desc_lo(smem_u32(v_img), kPanel);
      bool ok = true;
      for (int s = 0; s < slots && ok; ++s) ok = warp_wait(&bar.q_full[s], 0, err, kErrTimeoutFull);
      for (int i = 0; i <= units && ok; ++i) {
        // S of unit i over P of unit i - 2, whose product was issued before
        if (i < units) {
          const int at = i % S::units;
          ok = warp_wait(&bar.k_full[at], (i / S::units) & 1, err, kErrTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t kd = k_desc + at * (S::unit >> 4);
          for (int s = 0; s < slots; ++s) {
            const int buf = s * 2 + (i & 1);
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
              const uint32_t b_lo = kd + (e >> 2) * (kPanel >> 4) + (e & 3) * (32 >> 4);
              if constexpr (S::q_tmem)
                mma_ts(leader, tm + buf * 64, tm + S::q_col + s * (D / 2) + 8 * e, b_lo, id_qk, e != 0);
              else
                mma_ss(leader, tm + buf * 64, q_desc + s * (S::q_tile >> 4) + (e >> 2) * (kQPanel >> 4) + (e & 3) * (32 >> 4),
                       b_lo, id_qk, e != 0);
            }
            commit(leader, smem_u32(&bar.s_full[buf]));
            arrive(leader, smem_u32(&bar.s_full[buf]));
            if (s == slots - 1) commit(leader, smem_u32(&bar.k_empty[at]));
          }
        }
        if (i > 0) {
          const int at = (i - 1) % S::units;
          ok = warp_wait(&bar.v_full[at], ((i - 1) / S::units) & 1, err, kErrTimeoutFull);
          const uint32_t vd = v_desc + at * (S::unit >> 4);
          for (int s = 0; s < slots && ok; ++s) {
            const int buf = s * 2 + ((i - 1) & 1);
            ok = warp_wait(&bar.p_full[buf], ((i - 1) >> 1) & 1, err, kErrTimeoutFull);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int e = 0; e < kKeys / 16; ++e)
              mma_ts(leader, tm + S::o_col + s * D, tm + buf * 64 + 8 * e, vd + e * (2048 >> 4), id_pv, i > 1 || e != 0);
            commit(leader, smem_u32(&bar.pv_done[s]));
            if (s == slots - 1) commit(leader, smem_u32(&bar.v_empty[at]));
          }
        }
      }
      if (!ok) {  // a wait gave up: nothing issued here may run on when tensor memory is freed
        commit(leader, smem_u32(&bar.drained));
        warp_wait(&bar.drained, 0, err, kErrTimeoutOther);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, 512);
}

template <int D, int SLOTS>
cudaError_t prepare() {
  using S = Shape<D, SLOTS>;
  cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<D, SLOTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
  if (e != cudaSuccess) return e;
  cudaFuncAttributes at;
  if ((e = cudaFuncGetAttributes(&at, kv8_prompt_kernel<D, SLOTS>)) != cudaSuccess) return e;
  // the roles' registers come out of what the launch has: more than that would be waited for without end
  if (at.numRegs != S::regs) return cudaErrorInvalidConfiguration;
  return cudaSuccess;
}

template <int D, int SLOTS>
cudaError_t run(const Kv8Attn& a) {
  using S = Shape<D, SLOTS>;
  const cudaError_t e = prepare<D, SLOTS>();
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(a.pages.heads) * a.chunks, a.seqs.batch, a.row_groups);
  kv8_prompt_kernel<D, SLOTS><<<grid, S::threads, S::smem, a.stream>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace kv8

void kv8_prompt_plan(Kv8Attn& a, int sms) {
  const long long rows = static_cast<long long>(a.seqs.tokens) * a.group;
  a.tile_rows = a.head_dim == 256 || rows <= 128 ? 128 : 256;
  a.row_groups = static_cast<int>((rows + a.tile_rows - 1) / a.tile_rows);
  const long long tiles = static_cast<long long>(a.seqs.batch) * a.pages.heads * a.row_groups;
  long long span = a.max_len;
  if (a.window) span = std::min(span, static_cast<long long>(a.window) + a.tile_rows / a.group + 32);
  span = std::max(span, 1ll);
  // where the row groups do not fill the SMs, the keys are cut, into 512 at the least
  const long long want = std::max(1ll, std::min(sms / tiles, span / 512));
  const long long chunk = ((span + want - 1) / want + kv8::kKeys - 1) / kv8::kKeys * kv8::kKeys;
  a.chunk = static_cast<int>(chunk);
  a.chunks = static_cast<int>((span + chunk - 1) / chunk);
}

cudaError_t launch_kv8_prompt(const Kv8Attn& a) {
  switch (a.head_dim * 1000 + a.tile_rows) {
    case 64128: return kv8::run<64, 1>(a);
    case 64256: return kv8::run<64, 2>(a);
    case 128128: return kv8::run<128, 1>(a);
    case 128256: return kv8::run<128, 2>(a);
    case 256128: return kv8::run<256, 1>(a);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t kv8_prompt_error(int* code, cudaStream_t stream) { return kv8_take_error(&kv8::g_error, code, stream); }

}  // namespace qhtp
