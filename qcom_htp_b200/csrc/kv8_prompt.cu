// Attention of many query rows (prompts, pieces of prompts) over the 8-bit paged KV cache, on tcgen05.
//
// The mathematics is kv8_decode.cu's: exponents t = q . ck * (scale log2(e) sk) + log2(sv), outputs
// sum 2^(t - m) cv / sum 2^(t - m) / sv, the int8 codes as f16 operands, V's scale in the exponent.
//
// A CTA owns a tile of 128 query rows (the tokens and heads of one kv head's group, packed) and walks over the
// keys 64 at a time (head_dim 256, and groups of at most 128 rows; kv8_prompt2.cu has two tiles a CTA for the others):
//   copying warps bring codes from the paged cache by bulk copies into staging buffers (a 16-key group of a head is
//     contiguous in its block), and one the blocks' scales;
//   K and V converters (a warpgroup each) write them as f16 into 128-byte-swizzled images [key][64 head_dim], two to
//     four units ahead: K-major for Q K^T, and the same bytes MN-major for P V;
//   one warp issues the MMAs: S = Q K^T into tensor memory, O += P V with P read from tensor memory;
//   two softmax warpgroups, two threads per row with 32 keys each: S from tensor memory, P back over it as f16.
// There are two S buffers, so that the softmax of one unit runs under the MMAs of its neighbours.  Q stands in tensor
// memory: an MMA of 64 columns then reads 2 KB of shared memory where it would read 6.
//
// m is raised, and O rescaled, only when a row's maximum has grown by more than 2^8: p, taken to m - kLift, then stays below
// 2^15, inside f16, and most units leave O alone.
//
// Measured: 2 prompts of up to 2500 tokens, 16 heads x 256 over 2: 93 us (640 TFLOP/s of visible pairs); 6 tokens of 28 heads x 128
// over 4 of each of 16 sequences of up to 4100 keys: 28 us.  A unit of 64 keys takes some 1600 cycles (head_dim 128) to 2500 (256):
// its MMAs 630 and 1260 (64 columns cost 47 cycles where they should 32), at head_dim 256 shared memory 1500 (codes in and
// out, images in, operands out: 192 KB), the way from S to P 1000.  A CTA starts 8 us before its first S: tables, codes and Q are
// chains of loads, and there is room for one CTA only.  Rows split between two slots that take the keys in turn, each with its
// own O (kv8_prompt2.cu's layout, 128 keys a tile) were no faster (65 us against 65 at 48 rows, 124 against 112 at 40 of 60
// sequences), for two parts to join instead of one.
#include <algorithm>

#include "kv8_prompt.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kKeys = 64;              // keys of a unit
constexpr int kPanel = kKeys * 128;    // bytes of a [64 keys][64 f16] swizzled image

struct Barriers {
  uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full[2], pv_done, o_full, drained, staged[2][4], taken[2][4];
};

struct Small {
  float4 scale[8][4];     // (c, log2 w, 1 / w, care) of a unit's 16-key groups, eight units deep
  // [turn][half][row]: a half row's maximum, at the end its sum; at the start, before half[1] is in use, half[1][0] has
  // the rows' factors
  float half[2][2][128];
  Barriers bar;
  uint32_t tmem;
  Place place;            // for the end: what the block is about takes no registers until then
};

template <int D>
struct Shape {
  static constexpr int panels = D / 64;
  static constexpr int unit = panels * kPanel;                  // 64 keys of K or V
  static constexpr int k_units = D == 256 ? 2 : 4, v_units = D == 256 ? 3 : 4;
  static constexpr int depth = D == 256 ? 2 : 4;                // staging buffers of K, and of V
  static constexpr int staging = kKeys * D;                     // one of them
  static constexpr int q_tile = panels * kQPanel;
  // Q's image on its way to tensor memory: where there is no room for it, it passes through V's last units
  static constexpr int q_smem = D == 256 ? 0 : q_tile;
  static constexpr int data = q_smem + (k_units + v_units) * unit + 2 * depth * staging;
  static constexpr int smem = data + sizeof(Small);
  static_assert(smem <= 227 * 1024, "shared memory");
  static_assert(q_smem != 0 || q_tile <= (v_units - 1) * unit, "Q in V's units");
  static constexpr int threads = 640;
  // registers of a thread: at launch (the most that the threads leave room for), and by role
  static constexpr int regs = 96, softmax_regs = 112, convert_regs = 96, issue_regs = 64;
  static_assert(2 * softmax_regs + 2 * convert_regs + issue_regs <= 5 * regs, "registers");
  // tensor memory columns: two S buffers of 64 from 0, Q, O
  static constexpr int q_col = 128, o_col = 256;
  static_assert(q_col + D / 2 <= o_col && o_col + D <= 512, "tensor memory");
};

__device__ int g_error;  // a wait that gave up leaves its code here

// FIT: cut by fit_place, else on the plan's grid.  Two kernels, since that code costs the other one registers.
template <int D, bool FIT>
__global__ void __launch_bounds__(Shape<D>::threads, 1) kv8_prompt_kernel(const Kv8Attn a) {
  using S = Shape<D>;
  int* const err = &g_error;
  extern __shared__ __align__(1024) uint8_t smem[];
  Small& small = *reinterpret_cast<Small*>(smem + S::data);
  Barriers& bar = small.bar;
  float(&s_half)[2][2][128] = small.half;
  float(&s_down)[128] = small.half[1][0];
  float4(&s_scale)[8][4] = small.scale;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Place place;
  if constexpr (FIT) {
    if (!fit_place(a, blockIdx.x, reinterpret_cast<int2*>(smem), place)) return;
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
  const int R = T * a.group, r0 = place.rg * 128;
  if (r0 >= R) return;
  const int r1 = min(R, r0 + 128);
  const int len = seq_length(a, b);
  const Span all = row_span(a, len, T, r0, r1);
  const Span keys = chunk_span(place, all);
  if (threadIdx.x == 0) small.place = place;
  const int units = keys.lo < keys.hi ? (keys.hi - keys.lo + kKeys - 1) / kKeys : 0;
  if (units == 0 && place.chunk > 0) return;

  uint8_t* const k_img = smem + S::q_smem;
  uint8_t* const v_img = k_img + S::k_units * S::unit;
  uint8_t* const stage_img = v_img + S::v_units * S::unit;
  uint8_t* const q_img = S::q_smem ? smem : v_img + S::unit;

  constexpr int kConvK = 8, kConvV = 12, kMma = 16, kCopyK = 17, kCopyV = 18, kScale = 19;  // first warps of the roles
  if (warp == kMma) {
    tmem_alloc(&small.tmem, 512);
    if (lane == 0) {
      for (int i = 0; i < 4; ++i) {
        mbar_init(&bar.k_full[i], 5);  // the converter warps, and the one that brings the scales
        mbar_init(&bar.v_full[i], 4);
        mbar_init(&bar.k_empty[i], 1);
        mbar_init(&bar.v_empty[i], 1);
        for (int v = 0; v < 2; ++v) mbar_init(&bar.staged[v][i], 1), mbar_init(&bar.taken[v][i], 4);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bar.s_full[i], 2);  // the MMAs, and the issuing thread's own arrival
        mbar_init(&bar.p_full[i], 256);
      }
      mbar_init(&bar.q_full, 256);
      mbar_init(&bar.pv_done, 1);
      mbar_init(&bar.o_full, 1);
      mbar_init(&bar.drained, 1);
      fence_barrier_init();
    }
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = small.tmem;

  if (warp < kConvK) {
    // ------------------------------------------------------------------------------- softmax, two threads per row
    reg_alloc<S::softmax_regs>();
    const int half = warp >> 2, wq = warp & 3, in_tile = wq * 32 + lane, r = r0 + in_tile;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const uint32_t o_at = lanes + S::o_col + half * (D / 2);
    float m = -INFINITY, l = 0.0f;
    if (units > 0) {
      load_q<D, 16>(a, b, h, row0, r0, r1, q_img, s_down, warp, lane);
      named_barrier(1, 256);
      const float down = s_down[in_tile];
#pragma unroll 1
      for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
        uint32_t x[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = 4 * c + e;
          const uint4 v = *reinterpret_cast<const uint4*>(q_img + (at >> 3) * kQPanel + swizzled(in_tile, at & 7));
          x[4 * e] = v.x, x[4 * e + 1] = v.y, x[4 * e + 2] = v.z, x[4 * e + 3] = v.w;
        }
        tmem_st16(lanes + S::q_col + 16 * c, x);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar.q_full);
      const int p = len - T + r / a.group;
      const int row_hi = r >= r1 ? 0 : a.causal ? min(keys.hi, p + 1) : keys.hi, row_lo = a.window ? p - a.window + 1 : 0;
      // every row sees the keys [all_lo, all_hi)
      const int all_hi = a.causal ? min(keys.hi, len - T + r0 / a.group + 1) : keys.hi;
      const int all_lo = a.window ? len - T + (r1 - 1) / a.group - a.window + 1 : 0;
      bool ok = true;
      for (int i = 0; i < units; ++i) {
        const int buf = i & 1;
        const uint32_t s_at = lanes + buf * 64 + half * 32;
        // after a wait that gave up the rows are lost, but every warp still passes every named barrier
        ok = ok && warp_wait(&bar.s_full[buf], (i >> 1) & 1, err, kErrTimeoutAccum);
        tc_fence_after();
        uint32_t x[32], w[16];
        tmem_ld32(s_at, x);
        const int key0 = keys.lo + i * kKeys, col0 = key0 + half * 32;
        const View k{&s_scale[i & 7][2 * half], down, row_lo - col0, row_hi - col0};
        const bool careful = key0 + kKeys > all_hi || key0 < all_lo || s_scale[i & 7][0].w != 0.0f;
        tmem_ld_wait();
        pin(x);
        float top = careful ? row_max<true>(k, 0, x, m) : row_max<false>(k, 0, x, m);
        s_half[buf][half][in_tile] = top;
        named_barrier(2 + wq, 64);  // the two warps that share rows
        top = fmaxf(top, s_half[buf][half ^ 1][in_tile]);
        // raise m where it pays; rows of a warp move together, and its two halves alike
        if (__any_sync(0xffffffffu, top > m + kGrow || (m == -INFINITY && top != -INFINITY))) {
          const float alpha = m == -INFINITY ? 0.0f : ex2(m - top);
          if (i > 0) {
            ok = ok && warp_wait(&bar.pv_done, (i - 1) & 1, err, kErrTimeoutAccum);
            tc_fence_after();
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
        l = careful ? row_exp<true>(k, 0, x, base, l, w) : row_exp<false>(k, 0, x, base, l, w);
        tmem_st16(s_at, w);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar.p_full[buf]);
      }
      // a barrier of its own: pv_done may be one or two phases ahead of what this warp has seen, or at its end, and a parity
      // does not tell them apart
      if (ok) warp_wait(&bar.o_full, 0, err, kErrTimeoutAccum);
      tc_fence_after();
    }
    // the row's sum, and each half's columns of it
    s_half[units & 1][half][in_tile] = l;
    named_barrier(1, 256);
    l = s_half[units & 1][0][in_tile] + s_half[units & 1][1][in_tile];
    const float base = (m == -INFINITY ? 0.0f : m) - kLift;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long part0 = small.place.part + wq * 32, part = part0 + lane;
    // K's images are free: every S has been computed.  Rows of head_dim 64 are one piece, which the first half's warp takes.
    if (D > 64 || half == 0)
      rows_out<D, (D > 64 ? D / 2 : 64)>(a, b, h, row0, r0 + wq * 32, r1, part0, units == 0, o_at, D > 64 ? half * (D / 2) : 0, inv,
                                         small.place.chunks == 1, smem_u32(k_img) + warp * 4096, lane);
    const bool live = r < r1 && half == 0;
    if (live && small.place.chunks > 1) {
      float* ml = a.part + part_rows(a) * D + 2 * part;
      ml[0] = base, ml[1] = l;
    } else if (live && a.lse != nullptr) {
      const int t = r / a.group, head = h * a.group + r - t * a.group;
      const long long at = (a.seqs.start ? row0 : static_cast<long long>(b) * a.seqs.tokens) + t;
      a.lse[at * a.q_heads + head] = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.693147180559945309f;
    }
  } else if (warp < kMma) {
    // ------------------------------------------------------------------------------- codes to f16 images
    reg_free<S::convert_regs>();
    constexpr int kStep = 128 / (D / 8), kSteps = kKeys / kStep;
    const bool is_v = warp >= kConvV;
    const int t = threadIdx.x - (is_v ? kConvV : kConvK) * 32;
    // A thread has chunk c (eight codes, 16 bytes as f16) of the rows row, row + kStep, ...: loads and stores of a
    // warp are whole rows, without bank conflicts.
    const int c = t % (D / 8), row = t / (D / 8);
    const uint32_t from = smem_u32(stage_img) + (is_v ? S::depth * S::staging : 0) + row * D + c * 8;
    const uint32_t to = smem_u32(is_v ? v_img : k_img) + (c >> 3) * kPanel + swizzled(row, c & 7);
    uint64_t* const full = is_v ? bar.v_full : bar.k_full;
    uint64_t* const empty = is_v ? bar.v_empty : bar.k_empty;
    const int ring = is_v ? S::v_units : S::k_units;
    int at = 0, turn = 0;  // unit i % ring of the images, and i / ring
    for (int i = 0; i < units; ++i) {
      const int st = i % S::depth;
      if (!warp_wait(&bar.staged[is_v][st], (i / S::depth) & 1, err, kErrTimeoutFull)) break;
      uint2 raw[kSteps];
#pragma unroll
      for (int e = 0; e < kSteps; ++e) raw[e] = lds64(from + st * S::staging + e * kStep * D);
      if (turn > 0 && !warp_wait(&empty[at], (turn - 1) & 1, err, kErrTimeoutEmpty)) break;
      if (S::q_smem == 0 && is_v && i == 1 && !warp_wait(&bar.q_full, 0, err, kErrTimeoutEmpty)) break;  // Q has passed
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
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[at]);
        // only now: an arrival does not wait for loads before it whose values nothing has used, and the next copy would
        // overtake them
        mbar_arrive(&bar.taken[is_v][st]);
      }
      if (++at == ring) at = 0, ++turn;
    }
  } else {
    reg_free<S::issue_regs>();
    const int bs_log2 = a.pages.bs_log2, bs = 1 << bs_log2;
    // block of the unit's 16-key group `lane` (of four); -1: none
    auto ids_of = [&](int i) {
      const int key = keys.lo + i * kKeys + 16 * (lane & 3);
      return i < units && key < keys.hi ? static_cast<int>(block_of(a.seqs, a.pages, b, key >> bs_log2)) : -1;
    };
    if (warp == kCopyK || warp == kCopyV) {
      // ----------------------------------------------------------------------------- codes to the staging buffers
      // The table's entries are read a unit ahead.  Groups that there are none of keep the codes that happen to be there:
      // they are hidden, or their scales are NaN.
      const int v = warp == kCopyV;
      const int8_t* const codes = v ? a.pages.v : a.pages.k;
      uint8_t* const stage = stage_img + v * S::depth * S::staging;
      int id_next = ids_of(0), i = 0;
      for (; i < units; ++i) {
        const int st = i % S::depth, id = id_next;
        id_next = ids_of(i + 1);
        if (i >= S::depth && !warp_wait(&bar.taken[v][st], ((i / S::depth) - 1) & 1, err, kErrTimeoutEmpty)) break;
        const bool there = lane < 4 && id >= 0;
        const int count = __popc(__ballot_sync(0xffffffffu, there));
        if (lane == 0) mbar_arrive_expect_tx(&bar.staged[v][st], count * 16 * D);
        __syncwarp();
        if (there) {
          const int slot = (keys.lo + i * kKeys + 16 * lane) & (bs - 1);
          bulk_load(stage + st * S::staging + lane * 16 * D,
                    codes + (((static_cast<long long>(id) * a.pages.heads + h) << bs_log2) + slot) * D, 16 * D,
                    &bar.staged[v][st]);
        }
      }
      // copies under way end before the block does, also where a wait gave up, here or in the converters that take them
      for (int n = max(0, i - S::depth); n < i; ++n)
        warp_wait(&bar.staged[v][n % S::depth], (n / S::depth) & 1, err, kErrTimeoutOther);
    } else if (warp == kScale) {
      // ----------------------------------------------------------------------------- scales
      int id_next = ids_of(1);
      RawScales sc = units > 0 ? raw_scales(a, ids_of(0), h) : RawScales{};
      for (int i = 0; i < units; ++i) {
        const RawScales next = raw_scales(a, id_next, h);
        id_next = ids_of(i + 2);
        const int at = i % S::k_units;
        if (i >= S::k_units && !warp_wait(&bar.k_empty[at], ((i / S::k_units) - 1) & 1, err, kErrTimeoutEmpty)) break;
        // .w: a group whose scales need care (zero, or not finite)
        const BlockScales f = fold_scales(a, sc);
        const bool odd = !(f.inv_w < kZeroTile) || !isfinite(f.c);
        const float care = __any_sync(0xffffffffu, odd) ? 1.0f : 0.0f;
        if (lane < 4) s_scale[i & 7][lane] = make_float4(f.c, f.log2_w, f.inv_w, care);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.k_full[at]);
        sc = next;
      }
    } else if (units > 0) {
      // ----------------------------------------------------------------------------- the MMAs
      constexpr uint32_t id_qk = idesc_f16(128, kKeys), id_pv = idesc_f16(128, D, 1);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), leader = elect_one();
      const uint32_t k_desc = desc_lo(smem_u32(k_img), 16), v_desc = desc_lo(smem_u32(v_img), kPanel);
      bool ok = warp_wait(&bar.q_full, 0, err, kErrTimeoutFull);
      for (int i = 0; i <= units && ok; ++i) {
        // S of unit i over P of unit i - 2, whose product was issued before
        if (i < units) {
          const int at = i % S::k_units;
          ok = warp_wait(&bar.k_full[at], (i / S::k_units) & 1, err, kErrTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t kd = k_desc + at * (S::unit >> 4);
#pragma unroll
          for (int e = 0; e < D / 16; ++e)
            mma_ts(leader, tm + (i & 1) * 64, tm + S::q_col + 8 * e, kd + (e >> 2) * (kPanel >> 4) + (e & 3) * (32 >> 4), id_qk,
                   e != 0);
          commit(leader, smem_u32(&bar.s_full[i & 1]));
          arrive(leader, smem_u32(&bar.s_full[i & 1]));
          commit(leader, smem_u32(&bar.k_empty[at]));
        }
        if (i > 0) {
          const int at = (i - 1) % S::v_units, buf = (i - 1) & 1;
          ok = warp_wait(&bar.v_full[at], ((i - 1) / S::v_units) & 1, err, kErrTimeoutFull) &&
               warp_wait(&bar.p_full[buf], ((i - 1) >> 1) & 1, err, kErrTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vd = v_desc + at * (S::unit >> 4);
#pragma unroll
          for (int e = 0; e < kKeys / 16; ++e)
            mma_ts(leader, tm + S::o_col, tm + buf * 64 + (e >> 1) * 32 + (e & 1) * 8, vd + e * (2048 >> 4), id_pv, i > 1 || e != 0);
          commit(leader, smem_u32(&bar.pv_done));
          if (i == units) commit(leader, smem_u32(&bar.o_full));
          commit(leader, smem_u32(&bar.v_empty[at]));
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
cudaError_t prepare() {
  using S = Shape<D>;
  cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<D, FIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
  if (e != cudaSuccess) return e;
  cudaFuncAttributes at;
  if ((e = cudaFuncGetAttributes(&at, kv8_prompt_kernel<D, FIT>)) != cudaSuccess) return e;
  // the roles' registers come out of what the launch has: more than that would be waited for without end
  if (at.numRegs != S::regs) return cudaErrorInvalidConfiguration;
  return cudaSuccess;
}

template <int D, bool FIT>
cudaError_t run_as(const Kv8Attn& a) {
  using S = Shape<D>;
  static std::atomic<bool> done[64];
  const cudaError_t e = once_per_device(done, prepare<D, FIT>);
  if (e != cudaSuccess) return e;
  const dim3 grid = FIT ? dim3(a.fit) : dim3(static_cast<unsigned>(a.pages.heads) * a.chunks, a.seqs.batch, a.row_groups);
  kv8_prompt_kernel<D, FIT><<<grid, S::threads, S::smem, a.stream>>>(a);
  return cudaGetLastError();
}

template <int D>
cudaError_t run(const Kv8Attn& a) {
  return a.fit ? run_as<D, true>(a) : run_as<D, false>(a);
}

}  // namespace
}  // namespace kv8

void kv8_prompt_plan(Kv8Attn& a, int sms) {
  constexpr long long kLeast = 256;
  const long long rows = static_cast<long long>(a.seqs.tokens) * a.group;
  auto span_of = [&](int tile_rows) {
    long long span = a.max_len;
    if (a.window) span = std::min(span, static_cast<long long>(a.window) + tile_rows / a.group + 32);
    return std::max(span, 1ll);
  };
  auto groups_of = [&](int tile_rows) { return (rows + tile_rows - 1) / tile_rows; };
  // Two tiles a CTA where they can fill the SMs, with the keys cut as finely as may be.  Measured: 8192 tokens of 32 heads
  // 612 us against 801 with one; 60 tokens over 1500 keys 31 us against 23.
  const long long wide = a.seqs.batch * a.pages.heads * groups_of(256) * std::max(1ll, span_of(256) / kLeast);
  a.tile_rows = a.head_dim == 256 || rows <= 128 || wide < sms ? 128 : 256;
  a.row_groups = static_cast<int>(groups_of(a.tile_rows));
  const long long span = span_of(a.tile_rows);
  a.chunks = 1;
  a.chunk = static_cast<int>((span + 127) / 128 * 128);
  if (span < 2 * kLeast) return;
  // row groups of all sequences: the most that there can be, and about how many
  const long long most = static_cast<long long>(a.seqs.batch) * a.row_groups * a.pages.heads;
  const long long about =
      a.seqs.start ? std::min(most, (a.seqs.total * a.group / a.tile_rows + (a.seqs.batch + 1) / 2) * a.pages.heads) : most;
  if (2 * most <= sms && a.seqs.batch <= kv8::kFitBatch) {
    a.fit = sms;
    a.chunk = kLeast;
    a.chunks = static_cast<int>(std::min(sms / most, span / kLeast));
  } else if (span >= 4096 && about > sms && 2 * about <= 3 * sms) {
    // Three waves of half the keys are less than two of all, and over this many keys by more than the join costs.  Measured:
    // 160 row groups of 256 over 8000 keys 320 us whole, 280 in two; 176 of 128 (head_dim 256) over 4064 142 and 149.
    a.chunk = static_cast<int>((span / 2 + 127) / 128 * 128);
    a.chunks = 2;
  }
}

cudaError_t launch_kv8_prompt(const Kv8Attn& a) {
  switch (a.head_dim) {
    case 64: return kv8::run<64>(a);
    case 128: return kv8::run<128>(a);
    case 256: return kv8::run<256>(a);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t kv8_prompt_word(int** word) { return cudaGetSymbolAddress(reinterpret_cast<void**>(word), kv8::g_error); }

}  // namespace qhtp
