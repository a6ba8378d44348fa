// Device pieces shared by the tcgen05 attention kernels (kv8_prompt.cu, kv8_prompt2.cu).
#pragma once
#include "kv8.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kQPanel = 128 * 128;     // bytes of a [128 rows][64 f16] image of Q
constexpr float kGrow = 8.0f;          // log2 of how far p may pass 2^kLift before m follows
static_assert(kGrow + kLift <= 15.0f, "p and its rounding stay inside f16");

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
// (x * b + c, y * b + c) in one instruction
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
// Keeps uses of what tcgen05.ld wrote behind the wait for it: the wait itself does not name the registers.
template <int N>
__device__ __forceinline__ void pin(uint32_t (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(x[i]));
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
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
template <int D, int WARP_ROWS>
__device__ __forceinline__ void load_q(const Kv8Attn& a, int b, int h, long long row0, int r0, int r1, uint8_t* img,
                                       float* down_at, int warp, int lane) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // rows of a load
  constexpr int kBatch = D == 256 ? 16 : WARP_ROWS / kRows;  // loads in flight
  const int sub = lane / kLanes, c = lane % kLanes;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q.data) + b * a.q.batch_stride + row0 * a.q.token_stride +
                            static_cast<long long>(h) * a.group * a.q.head_stride + 8 * c;
  // token and head of the lane's next row
  int row = r0 + warp * WARP_ROWS + sub;
  int t = row / a.group, head = row - t * a.group;
#pragma unroll 1
  for (int base = 0; base < WARP_ROWS / kRows; base += kBatch) {
    uint4 w[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (row < r1) w[i] = __ldg(reinterpret_cast<const uint4*>(q + t * a.q.token_stride + head * a.q.head_stride));
      row += kRows;
      head += kRows;
      while (head >= a.group) head -= a.group, ++t;
    }
    uint32_t top[kBatch];
    if (a.bf16) {
      // bf16 magnitudes are ordered like their bits: the largest of the lane's, then of the row's.  A step of all rows at
      // a time: shuffles keep their order, and a row after the other would wait for each.
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        top[i] = __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu), __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top[i] = __vmaxu2(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = warp * WARP_ROWS + (base + i) * kRows + sub;
      float down = 1.0f;
      if (a.bf16) {
        float x[8];
        Vec<__nv_bfloat16>::load(w[i], x);
        float up;
        row_factor(__uint_as_float(max(top[i] & 0xffffu, top[i] >> 16) << 16), up, down);
        w[i] = make_uint4(pack_half2(x[0] * up, x[1] * up), pack_half2(x[2] * up, x[3] * up),
                          pack_half2(x[4] * up, x[5] * up), pack_half2(x[6] * up, x[7] * up));
      }
      *reinterpret_cast<uint4*>(img + (c >> 3) * kQPanel + swizzled(r, c & 7)) = w[i];
      if (c == 0) down_at[r] = down;
    }
  }
}

// A warp's 32 finished rows on their way out, 128 bytes of each at a time: a lane has a row in tensor memory, and stores of
// one row's 16 bytes each would take 32 lines at a time.  They go through 4 KB of shared memory instead, and leave as whole
// 128-byte pieces, four rows a store.
struct RowsOut {
  uint32_t stage;      // the warp's 4 KB
  uint8_t* to[8];      // this lane's 16 bytes of rows lane / 8, lane / 8 + 4, ...; null: not there
  // four 16-byte chunks of the lane's row, from chunk c0
  __device__ __forceinline__ void fill(int lane, int c0, const uint32_t* x) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) sts128(stage + swizzled(lane, c0 + c), x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
  }
  __device__ __forceinline__ void flush(int lane, int byte) const {
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint4 v = lds128(stage + swizzled(4 * k + (lane >> 3), lane & 7));
      if (to[k] != nullptr) *reinterpret_cast<uint4*>(to[k] + byte) = v;
    }
    __syncwarp();
  }
};

// COLS columns (a multiple of 64) of the warp's rows, from column col0 (O at o_at, or zeros): normalised to out, or as they
// are to the parts.  rw: the warp's first row of the group; part0: its part.
template <int D, int COLS>
__device__ __forceinline__ void rows_out(const Kv8Attn& a, int b, int h, long long row0, int rw, int r1, long long part0, bool zero,
                                         uint32_t o_at, int col0, float inv, bool whole, uint32_t stage, int lane) {
  RowsOut o;
  o.stage = stage;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int i = 4 * k + (lane >> 3), r = rw + i, t = r / a.group, head = h * a.group + r - t * a.group;
    uint8_t* p = whole ? reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(a.out.data) + b * a.out.batch_stride +
                                                    (row0 + t) * a.out.token_stride + head * a.out.head_stride + col0)
                       : reinterpret_cast<uint8_t*>(a.part + (part0 + i) * D + col0);
    o.to[k] = r < r1 ? p + (lane & 7) * 16 : nullptr;
  }
#pragma unroll 1
  for (int c = 0; c < COLS; c += 32) {
    uint32_t x[32];
    if (zero) {
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = 0;
    } else {
      tmem_ld32(o_at + c, x);
      tmem_ld_wait();
      pin(x);
    }
    if (whole) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float u = __uint_as_float(x[e]) * inv, v = __uint_as_float(x[e + 1]) * inv;
        x[e / 2] = a.bf16 ? Vec<__nv_bfloat16>::pack(u, v) : pack_half2(u, v);
      }
      o.fill(lane, (c & 32) / 8, x);
      if (c & 32) o.flush(lane, 2 * (c - 32));
    } else {
      o.fill(lane, 0, x);
      o.fill(lane, 4, x + 16);
      o.flush(lane, 4 * c);
    }
  }
}

// A row's view of some keys: their groups' constants, and the columns that the row sees.  CAREFUL below: there are
// columns that not every row sees, or a group whose scales are not plain.
struct View {
  const float4* scale;
  float down;
  int lo, hi;
};

// The largest exponent of the row in columns [col0, col0 + 32), or `top` where that is larger.
template <bool CAREFUL>
__device__ __forceinline__ float row_max(const View& k, int col0, const uint32_t (&x)[32], float top) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float4 sc = k.scale[col0 / 16 + c];
    const uint32_t* const v = &x[16 * c];
    if constexpr (CAREFUL) {
      float best = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = col0 + 16 * c + e;
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

// p of columns [col0, col0 + 32) as f16 pairs into w; returns l with the row's sum added.
template <bool CAREFUL>
__device__ __forceinline__ float row_exp(const View& k, int col0, const uint32_t (&x)[32], float base, float l, uint32_t (&w)[16]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float4 sc = k.scale[col0 / 16 + c];
    const uint32_t* const v = &x[16 * c];
    uint32_t* const to = &w[8 * c];
    const float f = sc.x * k.down, off = sc.y - base;
    float2 sum[2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      float2 t = fma2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), f, off);
      t.x = ex2(t.x), t.y = ex2(t.y);
      if constexpr (CAREFUL) {
        const int col = col0 + 16 * c + e;
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

}  // namespace
}  // namespace kv8
}  // namespace qhtp
