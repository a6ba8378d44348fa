// Attention of many query rows, two tiles of 128 rows a CTA (head_dim 64 and 128); the mathematics and the roles are
// kv8_prompt.cu's, the cut is another:
//   keys come 128 at a time, because an MMA of 64 columns takes 47 cycles or more where one of 128 takes 64;
//   each tile has one S buffer (tensor memory is full with two S and two O of head_dim 128), so the two tiles take turns:
//     the softmax of one runs under the MMAs of the other;
//   the time from S to P is therefore what counts, and a row is shared by two threads, 64 columns each: four softmax
//     warpgroups, so that a scheduler has four warps to hide latencies with.  They exchange their maxima once a tile;
//   one warpgroup converts both K and V.
//
// Measured: 8192 tokens of 32 heads x 128 over 8, causal, 0.60 to 0.65 ms (850 to 910 TFLOP/s of visible pairs; 0.80 ms in
// kv8_prompt.cu's kernel); 1000-token pieces of 3 sequences, 24 heads x 64 over 8, a window of 4096 keys: 133 us (330).  A tile of
// 128 keys takes some 4500 cycles for both slots: their MMAs 2050 (head_dim 64: 1540), the exponentials 2050 (16 a cycle), and each
// slot's chain from S over the maxima, the exchange and the exponentials to P, 2300, in which the other slot's MMAs fit.
// No faster: exponentials by polynomial on the FMA pipe for a part of the keys, an issuing warp for each slot (708 us against
// 606), deeper staging, slots held apart by barriers.
#include <algorithm>

#include "kv8_prompt.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kTile = 128;                // keys of a tile
constexpr int kUnit = 64;                 // keys of a staging buffer
constexpr int kPanel2 = kTile * 128;      // bytes of a [128 keys][64 f16] swizzled image
constexpr int kStaged = 3;                // staging buffers

template <int D>
struct Shape2 {
  static constexpr int tile = D / 64 * kPanel2;                 // K or V
  static constexpr int q_tile = D / 64 * kQPanel;
  static constexpr int staging = kUnit * D;                     // a staging buffer
  static constexpr int smem = 2 * q_tile + 4 * tile + kStaged * staging + 1024;
  static constexpr int threads = 768;
  // registers of a thread: at launch, and by role (four softmax warpgroups, one of converters, one with the issuing warp)
  static constexpr int regs = 80, softmax_regs = 96, convert_regs = 48, mma_regs = 48;
  static_assert(4 * softmax_regs + convert_regs + mma_regs <= 6 * regs, "registers");
  // tensor memory columns: S of the two tiles, O of the two, Q of the two where there is room
  static constexpr bool q_tmem = D == 64;
  static constexpr int o_col = 256, q_col = o_col + 2 * D;
  static_assert(o_col + 2 * D <= 512 && (!q_tmem || q_col + D <= 512), "tensor memory");
};

struct Barriers2 {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], drained, staged[kStaged], taken[kStaged];
};

__device__ int g_error2;  // a wait that gave up leaves its code here

// FIT: cut by fit_place, else on the plan's grid.  Two kernels, since that code costs the other one registers.
template <int D, bool FIT>
__global__ void __launch_bounds__(Shape2<D>::threads, 1) kv8_prompt2_kernel(const Kv8Attn a) {
  using S = Shape2<D>;
  int* const err = &g_error2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers2 bar;
  __shared__ uint32_t s_tmem;
  __shared__ Place s_place;  // for the end: what the block is about takes no registers until then
  __shared__ float s_down[256];
  __shared__ float s_half[2][2][2][128];  // [turn][slot][half][row]: a half row's maximum, at the end its sum
  __shared__ float4 s_scale[4][8];        // (c, log2 w, 1 / w, care) of a tile's 16-key groups, four tiles deep
  static_assert(sizeof(Barriers2) + 1024 + 4096 + 512 + 4 + sizeof(Place) + S::smem <= 227 * 1024, "shared memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Place place;
  if constexpr (FIT) {
    if (!fit_place(a, blockIdx.x, reinterpret_cast<int2*>(smem_raw), place)) return;
  } else {
    // heads fastest, the longest row groups (the last of a causal sequence) first
    place.h = blockIdx.x / a.chunks, place.chunk = blockIdx.x - place.h * a.chunks, place.b = blockIdx.y;
    place.rg = a.row_groups - 1 - blockIdx.z;
    place.chunks = a.chunks, place.keys = a.chunk;
  }
  const int b = place.b, h = place.h;
  long long row0;
  const int T = seq_rows(a.seqs, b, row0);
  if constexpr (!FIT) place.part = part_row(a, b, row0, h, place.rg, place.chunk);
  const int R = T * a.group, r0 = place.rg * 256;
  if (r0 >= R) return;
  const int r1 = min(R, r0 + 256);
  const int len = seq_length(a, b);
  const Span all = row_span(a, len, T, r0, r1);
  const Span keys = chunk_span(place, all);
  if (threadIdx.x == 0) s_place = place;
  const int tiles = keys.lo < keys.hi ? (keys.hi - keys.lo + kTile - 1) / kTile : 0;
  if (tiles == 0 && place.chunk > 0) return;

  uint8_t* const q_img = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* const k_img = q_img + 2 * S::q_tile;
  uint8_t* const v_img = k_img + 2 * S::tile;
  uint8_t* const stage_img = v_img + 2 * S::tile;

  constexpr int kConv = 16, kMma = 20, kCopy = 21, kScale = 22;  // first warps of the roles
  if (warp == kMma) {
    tmem_alloc(&s_tmem, 512);
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bar.q_full[i], 256);
        mbar_init(&bar.k_full[i], 5);  // the converter warps, and the one that brings the scales
        mbar_init(&bar.v_full[i], 4);
        mbar_init(&bar.k_empty[i], 1);
        mbar_init(&bar.v_empty[i], 1);
        mbar_init(&bar.s_full[i], 2);  // the MMAs, and the issuing thread's own arrival
        mbar_init(&bar.p_full[i], 256);
        mbar_init(&bar.o_full[i], 1);
      }
      for (int i = 0; i < kStaged; ++i) mbar_init(&bar.staged[i], 1), mbar_init(&bar.taken[i], 4);
      mbar_init(&bar.drained, 1);
      fence_barrier_init();
    }
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < kConv) {
    // ------------------------------------------------------------------------------- softmax, two threads per row
    reg_alloc<S::softmax_regs>();
    const int slot = warp >> 3, half = (warp >> 2) & 1, wq = warp & 3, in_tile = wq * 32 + lane, r = r0 + slot * 128 + in_tile;
    const int sr0 = r0 + slot * 128, sr1 = min(r1, sr0 + 128);  // the slot's rows (none: sr0 >= sr1)
    const uint32_t lanes = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const uint32_t s_at = lanes + slot * 128 + half * 64, o_at = lanes + S::o_col + slot * D + half * (D / 2);
    float m = -INFINITY, l = 0.0f;
    if (sr0 < sr1) {
      if (tiles > 0) {
        load_q<D, 16>(a, b, h, row0, sr0, sr1, q_img + slot * S::q_tile, s_down + slot * 128, half * 4 + wq, lane);
        named_barrier(1 + slot, 256);
        const float down = s_down[slot * 128 + in_tile];
        if constexpr (S::q_tmem) {  // each half row its half of the columns
          uint32_t x[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 v = *reinterpret_cast<const uint4*>(q_img + slot * S::q_tile + swizzled(in_tile, 4 * half + e));
            x[4 * e] = v.x, x[4 * e + 1] = v.y, x[4 * e + 2] = v.z, x[4 * e + 3] = v.w;
          }
          tmem_st16(lanes + S::q_col + slot * (D / 2) + 16 * half, x);
          tmem_st_wait();
          tc_fence_before();
        } else {
          fence_proxy_async_smem();
        }
        mbar_arrive(&bar.q_full[slot]);
        const int p = len - T + r / a.group;
        const int row_hi = r >= sr1 ? 0 : a.causal ? min(keys.hi, p + 1) : keys.hi, row_lo = a.window ? p - a.window + 1 : 0;
        // every row of the slot sees the keys [all_lo, all_hi)
        const int all_hi = a.causal ? min(keys.hi, len - T + sr0 / a.group + 1) : keys.hi;
        const int all_lo = a.window ? len - T + (sr1 - 1) / a.group - a.window + 1 : 0;
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
          // after a wait that gave up the rows are lost, but every warp still passes every named barrier
          ok = ok && warp_wait(&bar.s_full[slot], j & 1, err, kErrTimeoutAccum);
          tc_fence_after();
          const int key0 = keys.lo + j * kTile;
          const int col0 = key0 + half * 64;
          const View k{&s_scale[j & 3][4 * half], down, row_lo - col0, row_hi - col0};
          const bool careful = key0 + kTile > all_hi || key0 < all_lo || s_scale[j & 3][0].w != 0.0f;
          // the row's maximum: of this half, then of both
          float top = m;
          uint32_t x[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tmem_ld32(s_at + 32 * c, x);
            tmem_ld_wait();
            pin(x);
            top = careful ? row_max<true>(k, 32 * c, x, top) : row_max<false>(k, 32 * c, x, top);
          }
          s_half[j & 1][slot][half][in_tile] = top;
          named_barrier(3 + 4 * slot + wq, 64);  // the two warps that share rows
          top = fmaxf(top, s_half[j & 1][slot][half ^ 1][in_tile]);
          // raise m where it pays; rows of a warp move together, and its two halves alike.  S of this tile came after the
          // product of the last, so O stands still.
          if (__any_sync(0xffffffffu, top > m + kGrow || (m == -INFINITY && top != -INFINITY))) {
            const float alpha = m == -INFINITY ? 0.0f : ex2(m - top);
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
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
          const float base = (m == -INFINITY ? 0.0f : m) - kLift;
          // p of 32 keys over the first half of their own columns of S; the last ones are still in x
#pragma unroll
          for (int c = 1; c >= 0; --c) {
            uint32_t w[16];
            if (c == 0) {
              tmem_ld32(s_at, x);
              tmem_ld_wait();
              pin(x);
            }
            l = careful ? row_exp<true>(k, 32 * c, x, base, l, w) : row_exp<false>(k, 32 * c, x, base, l, w);
            tmem_st16(s_at + 32 * c, w);
          }
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&bar.p_full[slot]);
        }
        if (ok) warp_wait(&bar.o_full[slot], 0, err, kErrTimeoutAccum);
        tc_fence_after();
      }
      // the row's sum, and each half's columns of it
      s_half[tiles & 1][slot][half][in_tile] = l;
      named_barrier(1 + slot, 256);
      l = s_half[tiles & 1][slot][0][in_tile] + s_half[tiles & 1][slot][1][in_tile];
      const float base = (m == -INFINITY ? 0.0f : m) - kLift;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int rw = sr0 + wq * 32;
      const long long part0 = s_place.part + slot * 128 + wq * 32, part = part0 + lane;
      // K's images are free: every S has been computed.  Rows of
      // head_dim 64 are one piece, which the first half's warp takes.
      if (D == 128 || half == 0)
        rows_out<D, 64>(a, b, h, row0, rw, sr1, part0, tiles == 0, o_at, half * 64, inv, s_place.chunks == 1,
                        smem_u32(k_img) + (D == 128 ? warp : slot * 4 + wq) * 4096, lane);
      const bool live = r < sr1;
      if (half == 0 && live) {
        if (s_place.chunks > 1) {
          float* ml = a.part + part_rows(a) * D + 2 * part;
          ml[0] = base, ml[1] = l;
        } else if (a.lse != nullptr) {
          const int t = r / a.group, head = h * a.group + r - t * a.group;
          const long long at = (a.seqs.start ? row0 : static_cast<long long>(b) * a.seqs.tokens) + t;
          a.lse[at * a.q_heads + head] = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.693147180559945309f;
        }
      }
    }
  } else if (warp < kMma) {
    // ------------------------------------------------------------------------------- codes to f16 images
    reg_free<S::convert_regs>();
    // Pieces of 64 keys in the order of their use: K's two of a tile, V's two, the next tile's.
    constexpr int kStep = 128 / (D / 8), kSteps = kUnit / kStep;
    const int t = threadIdx.x - kConv * 32;
    // A thread has chunk c (eight codes, 16 bytes as f16) of the rows row, row + kStep, ...: loads and stores of a
    // warp are whole rows, without bank conflicts, and the swizzle of its rows is one number (kStep is a multiple of 8).
    static_assert(kStep % 8 == 0, "swizzle");
    const int c = t % (D / 8), row = t / (D / 8);
    const uint32_t from = smem_u32(stage_img) + row * D + c * 8;
    const uint32_t to = smem_u32(k_img) + (c >> 3) * kPanel2 + swizzled(row, c & 7);
    bool ok = true;
    for (int n = 0; n < 4 * tiles && ok; ++n) {
      const int j = n >> 2, q = n & 3, st = j & 1, at = n % kStaged;
      if (!warp_wait(&bar.staged[at], (n / kStaged) & 1, err, kErrTimeoutFull)) break;
      uint2 raw[kSteps];
#pragma unroll
      for (int e = 0; e < kSteps; ++e) raw[e] = lds64(from + at * S::staging + e * kStep * D);
      if ((q & 1) == 0 && j >= 2)
        ok = warp_wait(q ? &bar.v_empty[st] : &bar.k_empty[st], ((j >> 1) - 1) & 1, err, kErrTimeoutEmpty);
      const uint32_t img = to + (q & 2 ? 2 * S::tile : 0) + st * S::tile + (q & 1) * (kUnit * 128);
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        uint32_t u[4];
        codes_to_half2(raw[e].x, u[0], u[1]);
        codes_to_half2(raw[e].y, u[2], u[3]);
        sts128(img + e * kStep * 128, u[0], u[1], u[2], u[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      // only now: an arrival does not wait for loads before it whose values nothing has used, and the next copy would
      // overtake them
      if (lane == 0) mbar_arrive(&bar.taken[at]);
      if ((q & 1) && lane == 0) mbar_arrive(q & 2 ? &bar.v_full[st] : &bar.k_full[st]);
    }
  } else {
    // ------------------------------------------------------------------------------- the MMAs
    reg_free<S::mma_regs>();
    const int bs_log2 = a.pages.bs_log2, bs = 1 << bs_log2;
    // block of the tile's 16-key group `lane` (of eight); -1: none
    auto ids_of = [&](int j) {
      const int key = keys.lo + j * kTile + 16 * (lane & 7);
      return j < tiles && key < keys.hi ? static_cast<int>(block_of(a.seqs, a.pages, b, key >> bs_log2)) : -1;
    };
    if (warp == kCopy) {
      // codes to the staging buffers, in the order of their use; the table's entries are read a tile ahead.  Groups that there
      // are none of keep the codes that happen to be there: they are hidden, or their scales are NaN.
      int id = -1, id_next = ids_of(0), n = 0;
      bool ok = true;
      for (; n < 4 * tiles; ++n) {
        const int j = n >> 2, u = n & 1, at = n % kStaged;
        if ((n & 3) == 0) id = id_next, id_next = ids_of(j + 1);
        if (n >= kStaged) ok = warp_wait(&bar.taken[at], ((n / kStaged) - 1) & 1, err, kErrTimeoutEmpty);
        if (!ok) break;
        const bool there = (lane >> 2) == u && id >= 0;
        const int count = __popc(__ballot_sync(0xffffffffu, there));
        if (lane == 0) mbar_arrive_expect_tx(&bar.staged[at], count * 16 * D);
        __syncwarp();
        if (there) {
          const int slot = (keys.lo + j * kTile + 16 * lane) & (bs - 1);
          bulk_load(stage_img + at * S::staging + (lane & 3) * 16 * D,
                    (n & 2 ? a.pages.v : a.pages.k) + (((static_cast<long long>(id) * a.pages.heads + h) << bs_log2) + slot) * D,
                    16 * D, &bar.staged[at]);
        }
      }
      // copies under way end before the block does, also where a wait gave up, here or in the converters that take them
      for (int i = max(0, n - kStaged); i < n; ++i)
        warp_wait(&bar.staged[i % kStaged], (i / kStaged) & 1, err, kErrTimeoutOther);
    } else if (warp == kScale) {
      int id_next = ids_of(1);
      RawScales sc = tiles > 0 ? raw_scales(a, ids_of(0), h) : RawScales{};
      for (int j = 0; j < tiles; ++j) {
        const RawScales next = raw_scales(a, id_next, h);
        id_next = ids_of(j + 2);
        if (j >= 2 && !warp_wait(&bar.k_empty[j & 1], ((j >> 1) - 1) & 1, err, kErrTimeoutEmpty)) break;
        // .w: a group whose scales need care (zero, or not finite)
        const BlockScales f = fold_scales(a, sc);
        const bool odd = !(f.inv_w < kZeroTile) || !isfinite(f.c);
        const float care = __any_sync(0xffffffffu, odd) ? 1.0f : 0.0f;
        if (lane < 8) s_scale[j & 3][lane] = make_float4(f.c, f.log2_w, f.inv_w, care);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.k_full[j & 1]);
        sc = next;
      }
    } else if (warp == kMma && tiles > 0) {
      const int slots = r0 + 128 < r1 ? 2 : 1;
      constexpr uint32_t id_qk = idesc_f16(128, kTile), id_pv = idesc_f16(128, D, 1);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), leader = elect_one();
      const uint32_t q_desc = desc_lo(smem_u32(q_img), 16), k_desc = desc_lo(smem_u32(k_img), 16),
                     v_desc = desc_lo(smem_u32(v_img), kPanel2);
      bool ok = true;
      for (int s = 0; s < slots && ok; ++s) ok = warp_wait(&bar.q_full[s], 0, err, kErrTimeoutFull);
      for (int j = 0; j <= tiles && ok; ++j) {
        for (int s = 0; s < slots; ++s) {
          if (j > 0) {
            const int st = (j - 1) & 1;
            ok = warp_wait(&bar.v_full[st], ((j - 1) >> 1) & 1, err, kErrTimeoutFull) &&
                 warp_wait(&bar.p_full[s], (j - 1) & 1, err, kErrTimeoutFull);
            if (!ok) break;
            tc_fence_after();
            const uint32_t vd = v_desc + st * (S::tile >> 4);
#pragma unroll
            for (int e = 0; e < kTile / 16; ++e)
              mma_ts(leader, tm + S::o_col + s * D, tm + s * 128 + (e >> 1) * 32 + (e & 1) * 8, vd + e * (2048 >> 4), id_pv,
                     j > 1 || e != 0);
            if (s == slots - 1) commit(leader, smem_u32(&bar.v_empty[st]));
            if (j == tiles) commit(leader, smem_u32(&bar.o_full[s]));
          }
          if (j < tiles) {  // S of the next tile over P: in order behind the product that reads it
            const int st = j & 1;
            ok = warp_wait(&bar.k_full[st], (j >> 1) & 1, err, kErrTimeoutFull);
            if (!ok) break;
            tc_fence_after();
            const uint32_t kd = k_desc + st * (S::tile >> 4);
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
              const uint32_t b_lo = kd + (e >> 2) * (kPanel2 >> 4) + (e & 3) * (32 >> 4);
              if constexpr (S::q_tmem)
                mma_ts(leader, tm + s * 128, tm + S::q_col + s * (D / 2) + 8 * e, b_lo, id_qk, e != 0);
              else
                mma_ss(leader, tm + s * 128, q_desc + s * (S::q_tile >> 4) + (e >> 2) * (kQPanel >> 4) + (e & 3) * (32 >> 4), b_lo,
                       id_qk, e != 0);
            }
            commit(leader, smem_u32(&bar.s_full[s]));
            arrive(leader, smem_u32(&bar.s_full[s]));
            if (s == slots - 1) commit(leader, smem_u32(&bar.k_empty[st]));
          }
        }
      }
      // nothing issued here may run on when tensor memory is freed: where a wait gave up, here or in the softmax warps, no one
      // else has waited for it
      commit(leader, smem_u32(&bar.drained));
      warp_wait(&bar.drained, 0, err, kErrTimeoutOther);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, 512);
}

template <int D, bool FIT>
cudaError_t prepare2() {
  using S = Shape2<D>;
  cudaError_t e = cudaFuncSetAttribute(kv8_prompt2_kernel<D, FIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
  if (e != cudaSuccess) return e;
  cudaFuncAttributes at;
  if ((e = cudaFuncGetAttributes(&at, kv8_prompt2_kernel<D, FIT>)) != cudaSuccess) return e;
  // the roles' registers come out of what the launch has: more than that would be waited for without end
  return at.numRegs == S::regs ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <int D, bool FIT>
cudaError_t run_as2(const Kv8Attn& a) {
  using S = Shape2<D>;
  static std::atomic<bool> done[64];
  const cudaError_t e = once_per_device(done, prepare2<D, FIT>);
  if (e != cudaSuccess) return e;
  const dim3 grid = FIT ? dim3(a.fit) : dim3(static_cast<unsigned>(a.pages.heads) * a.chunks, a.seqs.batch, a.row_groups);
  kv8_prompt2_kernel<D, FIT><<<grid, S::threads, S::smem, a.stream>>>(a);
  return cudaGetLastError();
}

template <int D>
cudaError_t run2(const Kv8Attn& a) {
  return a.fit ? run_as2<D, true>(a) : run_as2<D, false>(a);
}

}  // namespace
}  // namespace kv8

cudaError_t launch_kv8_prompt2(const Kv8Attn& a) { return a.head_dim == 64 ? kv8::run2<64>(a) : kv8::run2<128>(a); }

cudaError_t kv8_prompt2_word(int** word) { return cudaGetSymbolAddress(reinterpret_cast<void**>(word), kv8::g_error2); }

}  // namespace qhtp
