// Attention of few query rows (single tokens, drafted tokens) over the 8-bit paged KV cache.
//
// Per row:  t_j = q . ck_j * (scale log2(e) sk) + log2(sv),   p_j = 2^(t_j - m),   m the running maximum of t less kLift
//           out = sum_j p_j cv_j / sum_j p_j / sv,            lse = ln 2 (m + log2(sum_j p_j / sv))
// with ck, cv the int8 codes of key j and sk, sv the scales of its block.  V's scale enters the
// exponent, so the codes themselves are the tensor core's operands (int8 is exact in f16), a scale
// costs nothing per element, and since the maximum is taken over t the largest p is 2^kLift: p rounded to f16 is off by at
// most 2^-11 of itself, and a small one by 2^-32 of the largest.  Scores, maxima, sums and outputs are float32.
//
// Bound by memory: two bytes per key and element.  The keys of a (sequence, kv head) are cut into chunks
// over the grid, a CTA's four warps take 32 of them (16 at head_dim 256) in turn, and each warp keeps a ring of
// them in shared memory filled by TMA, so that the loads in flight do not hang on registers or on what the warp does.
// Measured: 2 sequences of 131072 keys, 8 kv heads x 128, 90 us (6.0 TB/s; 6.4 to 6.5 between the first loads and the last; the
// same with blocks of 16, 32, 64 and 128);
// 64 of 4000 on average 101 us (5.3 TB/s); 16 of 9500 on average, 2 x 256, 35 us (4.4 TB/s).  What is left is a CTA's start
// (some 4 us until its first keys arrive) and the last CTAs' end, and the join (3 to 5 us).
// Keys are the M side of the MMAs (m16n8k16, S^T = K Q^T and O^T = V^T P^T), so a group of eight query rows
// wastes nothing.  Which head_dim index a fragment's k stands for is free: a thread's 16 bytes of a key are its
// fragments, and with the swizzle that TMA applies neither K's nor V's reads have bank conflicts (V of head_dim 64: two ways).
#include <algorithm>

#include "kv8.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kWarps = 4;
constexpr int kSegBlocks = 256;  // blocks whose constants are in shared memory at a time

__device__ int g_error;          // a wait that gave up leaves its code here

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 matrix of 16-bit values held as one row pair per thread.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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

// NT groups of eight rows.
template <int D, int NT>
struct Ring {
  static constexpr int k16 = D == 256 || NT == 4 ? 1 : 2;        // 16-key groups of a step
  static constexpr int box = 16 * (D < 128 ? D : 128);           // bytes of a TMA box: 16 keys of a 128-byte panel
  static constexpr int panels = D == 256 ? 2 : 1;
  static constexpr int half = k16 * panels * box;                // K, or V, of a step
  static constexpr int stages = 16384 / (2 * half);              // 16 KB a warp
  static constexpr int smem = kWarps * stages * 2 * half + 1024;
  static_assert(2 * 8 * NT * (D + 4) * 4 <= smem - 1024, "the rows are joined in the rings' memory");
};

// FIT: cut by fit_place, else on the plan's grid.  Two kernels, since that code costs the other one registers.
template <int D, int NT, bool FIT>
__global__ void __launch_bounds__(kWarps * 32, NT == 4 ? 2 : 3)  // what the rings leave room for; of <256, 2> two
    kv8_decode_kernel(const Kv8Attn a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using Rg = Ring<D, NT>;
  constexpr int K16 = Rg::k16;
  constexpr int kRows = 8 * NT;
  constexpr int kQStride = D + 4;      // halves: rows 2 banks apart, so the 64-bit fragment reads do not collide
  constexpr int kOStride = D + 4;
  constexpr int KJ = D / 64;           // 16-byte pieces of a key in one thread
  constexpr int VW = D / 32;           // words of a V row in one thread
  constexpr int MT = D / 16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) __half s_q[kRows * kQStride];
  __shared__ float s_down[kRows], s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ int s_lo[kRows], s_hi[kRows];
  __shared__ int s_id[kSegBlocks];
  __shared__ float s_c[kSegBlocks], s_lw[kSegBlocks], s_iw[kSegBlocks];
  __shared__ uint64_t s_full[kWarps][Rg::stages];
  uint8_t* const ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float* const s_o = reinterpret_cast<float*>(ring);
  int* const err = &g_error;

  __shared__ Place s_place;  // for the end
  Place at;
  if constexpr (FIT) {
    if (!fit_place(a, blockIdx.x, reinterpret_cast<int2*>(ring), at)) return;
  } else {
    // chunks slowest: the first ones, which every sequence has whole, run first, and the remainders fill the end
    at.b = blockIdx.y, at.h = blockIdx.x / a.row_groups, at.rg = blockIdx.x - at.h * a.row_groups, at.chunk = blockIdx.z;
    at.chunks = a.chunks, at.keys = a.chunk;
  }
  const int b = at.b, h = at.h;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  long long row0;
  const int T = seq_rows(a.seqs, b, row0);
  const int R = T * a.group, r0 = at.rg * kRows;
  if (r0 >= R) return;
  const int r1 = min(R, r0 + kRows);
  const int len = seq_length(a, b);
  const Span all = row_span(a, len, T, r0, r1);
  const Span keys = chunk_span(at, all);
  if (threadIdx.x == 0) s_place = at;
  // an empty chunk leaves nothing; where every chunk is empty, the first one writes the rows
  if (keys.lo >= keys.hi && at.chunk > 0) return;
  // each row of the group sees the keys [all_lo, all_hi)
  const int all_hi = a.causal ? len - T + r0 / a.group + 1 : len;
  const int all_lo = a.window ? len - T + (r1 - 1) / a.group - a.window + 1 : 0;

  if (threadIdx.x == 0) tma_prefetch_desc(&map_k), tma_prefetch_desc(&map_v);
  if (lane < Rg::stages) mbar_init(&s_full[warp][lane], 1);
  fence_barrier_init();
  const uint32_t my_ring = smem_u32(ring) + warp * Rg::stages * 2 * Rg::half;
  uint32_t turn = 0;  // steps of this warp so far: stage turn % stages, phase turn / stages

  // q's rows are on their way (and, below, the first keys) before anything is done with them
  constexpr int E = D / 32, kMine = kRows / kWarps;  // elements of a lane, rows of a warp
  uint32_t qw[kMine][E / 2];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int row = r0 + warp + i * kWarps;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) qw[i][e] = 0;
    if (row < r1) {
      const int t = row / a.group;
      const uint16_t* src = static_cast<const uint16_t*>(a.q.data) + b * a.q.batch_stride + (row0 + t) * a.q.token_stride +
                            (static_cast<long long>(h) * a.group + row - t * a.group) * a.q.head_stride + lane * E;
      if constexpr (E == 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
        qw[i][0] = v.x, qw[i][1] = v.y, qw[i][2] = v.z, qw[i][3] = v.w;
      } else if constexpr (E == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
        qw[i][0] = v.x, qw[i][1] = v.y;
      } else {
        qw[i][0] = __ldg(reinterpret_cast<const uint32_t*>(src));
      }
    }
  }

  float acc[NT][MT][4], m[NT][2], l[NT][2], f[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) m[n][i] = -INFINITY, l[n][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][t][i] = 0.0f;
  }

  const int bs_log2 = a.pages.bs_log2, bs = 1 << bs_log2;
  // A segment may start inside a block.  It is whole steps, except for a span's last: a step's group that is not there is
  // not copied, and only the rows' own limits hide it, which lie at the end of the span and not at that of a segment.
  const long long seg_keys = (static_cast<long long>(kSegBlocks - 1) << bs_log2) & ~(16ll * K16 - 1);
  bool ok = true;
  for (long long seg0 = keys.lo; seg0 < keys.hi; seg0 += seg_keys) {
    const int seg = static_cast<int>(seg0), seg_hi = static_cast<int>(min(static_cast<long long>(keys.hi), seg0 + seg_keys));
    const int blk0 = seg >> bs_log2, nblk = ((seg_hi - 1) >> bs_log2) - blk0 + 1;
    for (int i = threadIdx.x; i < nblk; i += kWarps * 32)
      s_id[i] = static_cast<int>(block_of(a.seqs, a.pages, b, blk0 + i));
    __syncthreads();

    const int groups = (seg_hi - seg + 15) >> 4, tiles = (groups + K16 - 1) / K16;
    auto block_at = [&](int gi) { return ((seg + min(gi, groups - 1) * 16) >> bs_log2) - blk0; };
    // A lane per box: K and V, groups, panels.  A group that is not there (past the span's end), or that the table does not
    // map, is not copied: its codes are whatever the ring holds, and its keys are hidden or their scales NaN.
    auto copy = [&](int tile, uint32_t at) {
      constexpr int kBoxes = 2 * K16 * Rg::panels;
      const int st = at % Rg::stages, gi = tile * K16 + (lane / 2) % K16, panel = lane / (2 * K16);
      const int key = seg + gi * 16;
      const int id = lane < kBoxes && gi < groups ? s_id[block_at(gi)] : -1;
      const int n = __popc(__ballot_sync(0xffffffffu, id >= 0));
      if (lane == 0) mbar_arrive_expect_tx(&s_full[warp][st], n * Rg::box);
      __syncwarp();
      if (id >= 0) {
        const uint32_t to = my_ring + st * 2 * Rg::half + (lane & 1) * Rg::half + ((lane / 2) % K16 * Rg::panels + panel) * Rg::box;
        tma_load_3d(to, lane & 1 ? &map_v : &map_k, smem_u32(&s_full[warp][st]), panel * 128, key & (bs - 1),
                    static_cast<int>(id * static_cast<long long>(a.pages.heads) + h));
      }
    };
    const uint32_t turn0 = turn;
    for (int i = 0; i < Rg::stages; ++i)
      if (warp + i * kWarps < tiles) copy(warp + i * kWarps, turn0 + i);

    if (seg0 == keys.lo) {  // the rows of q, each scaled by a power of two into f16
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r = warp + i * kWarps, row = r0 + r;
        float x[E];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          if (a.bf16) {
            x[2 * e] = __uint_as_float(qw[i][e] << 16), x[2 * e + 1] = __uint_as_float(qw[i][e] & 0xffff0000u);
          } else {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&qw[i][e]));
            x[2 * e] = v.x, x[2 * e + 1] = v.y;
          }
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        float up, down;
        row_factor(__uint_as_float(top), up, down);
#pragma unroll
        for (int e = 0; e < E / 2; ++e)
          *reinterpret_cast<uint32_t*>(&s_q[r * kQStride + lane * E + 2 * e]) = pack_half2(x[2 * e] * up, x[2 * e + 1] * up);
        if (lane == 0) {
          const int p = len - T + row / a.group;
          s_down[r] = down;
          s_hi[r] = row < r1 ? (a.causal ? min(len, p + 1) : len) : 0;
          s_lo[r] = a.window ? p - a.window + 1 : 0;
        }
      }
    }
    for (int i = threadIdx.x; i < nblk; i += kWarps * 32) {
      const BlockScales s = fold_scales(a, raw_scales(a, s_id[i], h));
      s_c[i] = s.c, s_lw[i] = s.log2_w, s_iw[i] = s.inv_w;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) f[n][i] = s_down[8 * n + 2 * q4 + i];
    for (int tile = warp; tile < tiles && ok; tile += kWarps, ++turn) {
      ok = warp_wait(&s_full[warp][turn % Rg::stages], (turn / Rg::stages) & 1, err, kErrTimeoutFull);
      if (!ok) break;
      const uint32_t k_at = my_ring + (turn % Rg::stages) * 2 * Rg::half, v_at = k_at + Rg::half;
      // S^T = K Q^T
      float s[K16][NT][4];
#pragma unroll
      for (int i = 0; i < K16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][n][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        uint4 kr[K16][2];
#pragma unroll
        for (int i = 0; i < K16; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            const uint32_t box = k_at + (i * Rg::panels + (j >> 1)) * Rg::box;
            kr[i][r] = lds128(D == 64 ? box + row * 64 + ((q4 ^ ((row >> 1) & 3)) << 4)
                                      : box + row * 128 + (((2 * q4 + (j & 1)) ^ (row & 7)) << 4));
          }
        const int d0 = D == 64 ? 16 * q4 : 128 * (j >> 1) + 32 * q4 + 16 * (j & 1);  // head_dim of the piece
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          uint2 qf[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n)
            qf[n] = *reinterpret_cast<const uint2*>(&s_q[(8 * n + g) * kQStride + d0 + 4 * st]);
#pragma unroll
          for (int i = 0; i < K16; ++i) {
            const uint32_t w0 = reinterpret_cast<const uint32_t*>(&kr[i][0])[st];
            const uint32_t w1 = reinterpret_cast<const uint32_t*>(&kr[i][1])[st];
            uint32_t a0, a1, a2, a3;
            codes_to_half2(w0, a0, a2);
            codes_to_half2(w1, a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(s[i][n], a0, a1, a2, a3, qf[n].x, qf[n].y);
          }
        }
      }

      const int key0 = seg + tile * 16 * K16;
      const bool masked = key0 + 16 * K16 > all_hi || key0 < all_lo;
      float iw[K16], top[NT][2];
      bool zero[K16];  // a tile of V whose scale counts as zero
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n][0] = m[n][0], top[n][1] = m[n][1];
#pragma unroll
      for (int i = 0; i < K16; ++i) {
        const int bi = block_at(tile * K16 + i);
        const float c = s_c[bi], lw = s_lw[bi];
        iw[i] = s_iw[bi];
        zero[i] = iw[i] == kZeroTile;
        if (zero[i]) iw[i] *= 0.5f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float t = fmaf(s[i][n][e], c * f[n][e & 1], lw);
            if (masked) {
              const int key = key0 + 16 * i + g + 8 * (e >> 1), r = 8 * n + 2 * q4 + (e & 1);
              if (key >= s_hi[r] || key < s_lo[r]) t = -INFINITY;
            }
            s[i][n][e] = t;
            top[n][e & 1] = fmaxf(top[n][e & 1], t);
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], x));
          // a row that has seen nothing yet keeps the maximum -inf; its terms are 2^-inf against 0 (less kLift)
          const float base = top[n][i] == -INFINITY ? 0.0f : top[n][i];
          const float alpha = ex2(m[n][i] - base);
          m[n][i] = top[n][i];
          top[n][i] = base - kLift;
          l[n][i] *= alpha;
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[n][t][i] *= alpha, acc[n][t][i + 2] *= alpha;
        }
      uint32_t pb[K16][NT][2];
#pragma unroll
      for (int i = 0; i < K16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = ex2(s[i][n][e] - top[n][e & 1]);
            // a masked key adds nothing, whatever its block's scale is
            l[n][e & 1] += masked && p[e] == 0.0f ? 0.0f : p[e] * iw[i];
          }
          pb[i][n][0] = transpose8(zero[i] ? 0u : pack_half2(p[0], p[1]));
          pb[i][n][1] = transpose8(zero[i] ? 0u : pack_half2(p[2], p[3]));
        }
      // O^T += V^T P^T
#pragma unroll
      for (int i = 0; i < K16; ++i) {
        uint32_t vr[4][VW];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 2 * q4 + (x & 1) + 8 * (x >> 1);
          const uint32_t box = v_at + i * Rg::panels * Rg::box;
          if constexpr (D == 64) {
            const uint2 v = lds64(box + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
            vr[x][0] = v.x, vr[x][1] = v.y;
          } else {
#pragma unroll
            for (int w = 0; w < VW; w += 4) {
              const uint4 v = lds128(box + (w >> 2) * Rg::box + row * 128 + ((g ^ (row & 7)) << 4));
              vr[x][w] = v.x, vr[x][w + 1] = v.y, vr[x][w + 2] = v.z, vr[x][w + 3] = v.w;
            }
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t x[2][4];  // [key pair][element of the word]
#pragma unroll
          for (int kp = 0; kp < 2; ++kp) {
            const uint32_t u0 = vr[2 * kp][w] ^ 0x80808080u, u1 = vr[2 * kp + 1][w] ^ 0x80808080u;
            const uint32_t lo = prmt(u0, u1, 0x5140u), hi = prmt(u0, u1, 0x7362u);
            x[kp][0] = sub_1152(prmt(lo, 0x64646464u, 0x4140u));
            x[kp][1] = sub_1152(prmt(lo, 0x64646464u, 0x4342u));
            x[kp][2] = sub_1152(prmt(hi, 0x64646464u, 0x4140u));
            x[kp][3] = sub_1152(prmt(hi, 0x64646464u, 0x4342u));
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(acc[n][2 * w], x[0][0], x[0][1], x[1][0], x[1][1], pb[i][n][0], pb[i][n][1]);
            mma_f16(acc[n][2 * w + 1], x[0][2], x[0][3], x[1][2], x[1][3], pb[i][n][0], pb[i][n][1]);
          }
        }
      }
      __syncwarp();  // the stage is read
      if (tile + Rg::stages * kWarps < tiles) copy(tile + Rg::stages * kWarps, turn + Rg::stages);
    }
    if (!ok) {  // a wait gave up: what is under way lands before the block ends
      const uint32_t last = turn0 + (tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0);
      for (uint32_t i = 0; i < Rg::stages && turn + i < last; ++i)
        warp_wait(&s_full[warp][(turn + i) % Rg::stages], ((turn + i) / Rg::stages) & 1, err, kErrTimeoutOther);
      ok = false;
    }
    __syncthreads();  // the segment's constants, and the rings, are read
    if (!__syncthreads_and(ok)) break;
  }

  griddep_launch_dependents();
  // join the warps: every row's maximum, then the warps' rows beside one another in the rings' memory, or on top of
  // one another where they do not fit
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x);
      if (g == 0) s_m[warp][8 * n + 2 * q4 + i] = m[n][i], s_l[warp][8 * n + 2 * q4 + i] = l[n][i];
    }
  __syncthreads();
  constexpr int kArea = kRows * kOStride, kAreas = kWarps * kArea * 4 <= Rg::smem - 1024 ? kWarps : kWarps / 2;
  for (int w = 0; w < kWarps; w += kAreas) {
    if (warp >= w && warp < w + kAreas) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = 8 * n + 2 * q4 + i;
          float top = s_m[0][r];
#pragma unroll
          for (int x = 1; x < kWarps; ++x) top = fmaxf(top, s_m[x][r]);
          const float alpha = ex2(m[n][i] - (top == -INFINITY ? 0.0f : top));
          float* o = s_o + (warp - w) * kArea + r * kOStride;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int d = D == 64 ? 8 * g + 2 * t : 128 * (t >> 3) + 16 * g + 2 * (t & 7);
            float2 x = make_float2(acc[n][t][i] * alpha, acc[n][t][i + 2] * alpha);
            float2* to = reinterpret_cast<float2*>(o + d);
            if (w) x.x += to->x, x.y += to->y;
            *to = x;
          }
        }
    }
    __syncthreads();
  }

  const long long part = FIT ? s_place.part : part_row(a, b, row0, h, s_place.rg, s_place.chunk);
  const bool whole = s_place.chunks == 1;
  for (int i = threadIdx.x; i < kRows * (D / 8); i += kWarps * 32) {
    const int r = i / (D / 8), c = i - r * (D / 8), row = r0 + r;
    if (row >= r1) break;
    float top = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s_l[w][r] * ex2(s_m[w][r] - base);
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < kAreas; ++w) o[e] += s_o[w * kArea + r * kOStride + 8 * c + e];
    }
    if (whole) {
      write_row8(a, b, row0, row, h, 8 * c, o, sum, base - kLift);
    } else {
      float4* to = reinterpret_cast<float4*>(a.part + (part + r) * D + 8 * c);
      to[0] = make_float4(o[0], o[1], o[2], o[3]);
      to[1] = make_float4(o[4], o[5], o[6], o[7]);
      if (c == 0) {
        float* ml = a.part + part_rows(a) * D + 2 * (part + r);
        ml[0] = base - kLift, ml[1] = sum;
      }
    }
  }
}

// A row's parts: those that its attention kernel wrote, `step` rows apart.  None: the row is not there, or finished.
struct Parts {
  int b, h, row, n;
  long long row0, first, step;
  __device__ __forceinline__ long long at(int i) const { return first + i * step; }
};
__device__ __forceinline__ Parts parts_of(const Kv8Attn& a, int row) {
  Parts p{static_cast<int>(blockIdx.z), static_cast<int>(blockIdx.y), row, 0};
  const int T = seq_rows(a.seqs, p.b, p.row0);
  const int R = T * a.group, rg = row / a.tile_rows, r0 = rg * a.tile_rows, r1 = min(R, r0 + a.tile_rows);
  if (row >= R || rg >= a.row_groups) return p;
  int chunks = a.chunks, keys = a.chunk;
  if (a.fit) {
    const int4 cut = cuts_of(a)[p.b];
    if (cut.y == 1) return p;
    chunks = cut.y, keys = cut.z;
    p.first = static_cast<long long>(cut.x + cut.w - (rg + 1) * a.pages.heads + p.h) * a.tile_rows;
    p.step = static_cast<long long>(cut.w) * a.tile_rows;
  } else {
    p.first = part_row(a, p.b, p.row0, p.h, rg, 0);
    p.step = a.tile_rows;
  }
  p.first += row - r0;
  const Span s = row_span(a, seq_length(a, p.b), T, r0, r1);
  const long long span = s.hi - (s.lo & ~31);
  p.n = span <= 0 ? 1 : static_cast<int>(min(static_cast<long long>(chunks), (span + keys - 1) / keys));
  return p;
}

// The chunks of each row joined, few of them: D / 8 threads a row, each over all chunks, kFew at a time.  Up to kFew chunks
// (as many as equal lengths would have), else the kernel below: 2688 rows of 2 chunks 33.1 us with their attention, 41.3 by a CTA
// a row; 64 rows of 27 chunks 98.2 by a CTA a row, 103.9 by this one.
constexpr int kFew = 8;
template <int D>
__global__ void __launch_bounds__(128) kv8_combine_few_kernel(const Kv8Attn a) {
  constexpr int kLanes = D / 8, kPer = 128 / kLanes;
  griddep_wait();
  const int c = threadIdx.x % kLanes;
  const Parts p = parts_of(a, blockIdx.x * kPer + threadIdx.x / kLanes);
  if (p.n == 0) return;
  const float* const ml = a.part + part_rows(a) * D;
  float top = -INFINITY, sum = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < p.n; i0 += kFew) {
    float l[kFew], m[kFew];
    const float before = top;
#pragma unroll
    for (int i = 0; i < kFew; ++i) {
      const float2 v = i0 + i < p.n ? *reinterpret_cast<const float2*>(ml + 2 * p.at(i0 + i)) : make_float2(0.0f, 0.0f);
      m[i] = v.x, l[i] = v.y;
      if (v.y != 0.0f) top = fmaxf(top, v.x);
    }
    if (top == -INFINITY) continue;  // no key yet
    const float alpha = ex2(before - top);
    sum *= alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= alpha;
#pragma unroll
    for (int i = 0; i < kFew; ++i) {
      if (i0 + i >= p.n) break;
      const float4* x = reinterpret_cast<const float4*>(a.part + p.at(i0 + i) * D + 8 * c);
      const float4 u = x[0], v = x[1];
      const float f = l[i] != 0.0f ? ex2(m[i] - top) : 0.0f;
      sum = fmaf(l[i], f, sum);
      o[0] = fmaf(u.x, f, o[0]), o[1] = fmaf(u.y, f, o[1]), o[2] = fmaf(u.z, f, o[2]), o[3] = fmaf(u.w, f, o[3]);
      o[4] = fmaf(v.x, f, o[4]), o[5] = fmaf(v.y, f, o[5]), o[6] = fmaf(v.z, f, o[6]), o[7] = fmaf(v.w, f, o[7]);
    }
  }
  write_row8(a, p.b, p.row0, p.row, p.h, 8 * c, o, sum, top == -INFINITY ? 0.0f : top);
}

// The chunks of a row joined: a CTA a row.  Its threads take the chunks' maxima and sums at once, then each eight
// elements of every kGroups-th chunk; the groups are added up in their order.
template <int D>
__global__ void __launch_bounds__(256) kv8_combine_kernel(const Kv8Attn a) {
  constexpr int kLanes = D / 8, kGroups = 256 / kLanes, kWeights = 256;
  __shared__ float s_w[kWeights], s_top[8], s_sum[8];
  __shared__ float s_o[kGroups][D + 4];
  griddep_wait();
  const int t = threadIdx.x;
  const Parts p = parts_of(a, blockIdx.x);
  const int n = p.n;
  if (n == 0) return;
  const float* const ml = a.part + part_rows(a) * D;
  // the row's maximum over the chunks that saw a key of it
  float top = -INFINITY;
  for (int i = t; i < n; i += 256) {
    const float2 v = *reinterpret_cast<const float2*>(ml + 2 * p.at(i));
    if (v.y != 0.0f) top = fmaxf(top, v.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((t & 31) == 0) s_top[t >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, s_top[i]);
  if (top == -INFINITY) top = 0.0f;

  const int c = t % kLanes, group = t / kLanes;
  float sum = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int base = 0; base < n; base += kWeights) {
    const int m = min(kWeights, n - base);
    if (t < m) {
      const float2 v = *reinterpret_cast<const float2*>(ml + 2 * p.at(base + t));
      const float w = v.y != 0.0f ? ex2(v.x - top) : 0.0f;
      s_w[t] = w;
      sum = fmaf(v.y, w, sum);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = group; i < m; i += kGroups) {
      const float4* x = reinterpret_cast<const float4*>(a.part + p.at(base + i) * D + 8 * c);
      const float4 u = x[0], v = x[1];
      const float f = s_w[i];
      o[0] = fmaf(u.x, f, o[0]), o[1] = fmaf(u.y, f, o[1]), o[2] = fmaf(u.z, f, o[2]), o[3] = fmaf(u.w, f, o[3]);
      o[4] = fmaf(v.x, f, o[4]), o[5] = fmaf(v.y, f, o[5]), o[6] = fmaf(v.z, f, o[6]), o[7] = fmaf(v.w, f, o[7]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if ((t & 31) == 0) s_sum[t >> 5] = sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) s_o[group][8 * c + e] = o[e];
  __syncthreads();
  if (t >= kLanes) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += s_sum[i];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    o[e] = 0.0f;
    for (int i = 0; i < kGroups; ++i) o[e] += s_o[i][8 * t + e];
  }
  write_row8(a, p.b, p.row0, p.row, p.h, 8 * t, o, sum, top);
}

template <int D, int NT, bool FIT>
cudaError_t run_as(const Kv8Attn& a) {
  using Rg = Ring<D, NT>;
  CUtensorMap map[2];
  const uint64_t tiles = static_cast<uint64_t>(a.pages.num_blocks) * a.pages.heads;
  const CUtensorMapSwizzle swizzle = D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  for (int i = 0; i < 2; ++i)
    if (!make_tmap_tiles_u8(&map[i], i ? a.pages.v : a.pages.k, D, 1ull << a.pages.bs_log2, tiles, D < 128 ? D : 128, 16, swizzle))
      return cudaErrorInvalidValue;
  static std::atomic<bool> done[64];
  const cudaError_t e = once_per_device(done, [] {
    return cudaFuncSetAttribute(kv8_decode_kernel<D, NT, FIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Rg::smem);
  });
  if (e != cudaSuccess) return e;
  const dim3 grid = FIT ? dim3(a.fit) : dim3(static_cast<unsigned>(a.pages.heads) * a.row_groups, a.seqs.batch, a.chunks);
  kv8_decode_kernel<D, NT, FIT><<<grid, kWarps * 32, Rg::smem, a.stream>>>(a, map[0], map[1]);
  return cudaGetLastError();
}

template <int D, int NT>
cudaError_t run(const Kv8Attn& a) {
  return a.fit ? run_as<D, NT, true>(a) : run_as<D, NT, false>(a);
}

template <int D>
cudaError_t combine(const Kv8Attn& a) {
  const long long rows = static_cast<long long>(a.seqs.tokens) * a.group;
  const bool few = a.chunks <= kFew;
  const int per = few ? 128 / (D / 8) : 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + per - 1) / per), a.pages.heads, a.seqs.batch);
  cfg.blockDim = dim3(few ? 128 : 256);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return few ? cudaLaunchKernelEx(&cfg, kv8_combine_few_kernel<D>, a) : cudaLaunchKernelEx(&cfg, kv8_combine_kernel<D>, a);
}

}  // namespace
}  // namespace kv8

void kv8_decode_plan(Kv8Attn& a, int sms) {
  const long long rows = static_cast<long long>(a.seqs.tokens) * a.group;
  const int most = a.head_dim == 256 ? 16 : 32;
  a.tile_rows = rows <= 8 ? 8 : rows <= 16 || most == 16 ? 16 : 32;
  a.row_groups = static_cast<int>((rows + a.tile_rows - 1) / a.tile_rows);
  const long long tiles = static_cast<long long>(a.seqs.batch) * a.pages.heads * a.row_groups;
  // keys that a row group can see
  long long span = a.max_len;
  if (a.window) span = std::min(span, static_cast<long long>(a.window) + a.tile_rows + 31);
  span = std::max(span, 1ll);
  // Three CTAs fit an SM up to 16 rows, two with 32 (registers) and with 16 rows of head_dim 256 (shared memory), for which
  // the rules below, made for three, cut the keys into one and a half waves.  Where the row groups alone are many waves of those, chunks of kMost keys are short enough for
  // sequences of unlike lengths to share the SMs.  Else the keys are cut so that the CTAs are one whole wave (by the lengths:
  // fit_place).  Short spans are left whole: a CTA takes 512 keys in less time than a second kernel needs to join two parts.
  // Measured, 2 x 131072 keys: one wave 95.6 us, two 103.2, three 109.3, chunks of 2048 keys (2.3 waves) 110.
  // 500 keys whole 10.5 us, in two 13.2; 1500 keys in chunks of 128 12.7 us, of 256 14.7, whole 18.7.
  // By the lengths against chunks of the longest one's: 16 x up to 16000 keys of head_dim 256 42.4 us against 51.4, 24 x up to
  // 12000 of head_dim 64 31.4 against 41.4; all lengths alike, 16 x 8000, 57.1 against 54.5: what finding its place costs a CTA.
  // With more row groups than a wave holds: 64 x up to 8000 keys 108 us in chunks of 2048, 114 to 120 by the lengths
  // (two to four waves).
  constexpr long long kMost = 2048, kLeast = 128, kWhole = 768;
  const long long slots = 3ll * sms;
  long long n = 1;
  if (span > kWhole) {
    n = (span + kMost - 1) / kMost;
    if (n * tiles < 4 * slots) n = std::max(1ll, std::min(slots / tiles, span / kLeast));
    if (n * tiles <= slots && a.seqs.batch <= kv8::kFitBatch) {
      a.fit = static_cast<int>(slots);
      a.chunk = kLeast;
      a.chunks = static_cast<int>(n);
      return;
    }
  }
  n = std::min(n, 65535ll);  // grid.z
  const long long chunk = ((span + n - 1) / n + 127) / 128 * 128;
  a.chunk = static_cast<int>(chunk);
  a.chunks = static_cast<int>((span + chunk - 1) / chunk);
}

cudaError_t launch_kv8_decode(const Kv8Attn& a) {
  switch (a.head_dim * 100 + a.tile_rows) {
    case 6408: return kv8::run<64, 1>(a);
    case 6416: return kv8::run<64, 2>(a);
    case 6432: return kv8::run<64, 4>(a);
    case 12808: return kv8::run<128, 1>(a);
    case 12816: return kv8::run<128, 2>(a);
    case 12832: return kv8::run<128, 4>(a);
    case 25608: return kv8::run<256, 1>(a);
    case 25616: return kv8::run<256, 2>(a);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_kv8_combine(const Kv8Attn& a) {
  if (a.head_dim == 64) return kv8::combine<64>(a);
  if (a.head_dim == 128) return kv8::combine<128>(a);
  return kv8::combine<256>(a);
}

cudaError_t kv8_decode_word(int** word) { return cudaGetSymbolAddress(reinterpret_cast<void**>(word), kv8::g_error); }

}  // namespace qhtp
