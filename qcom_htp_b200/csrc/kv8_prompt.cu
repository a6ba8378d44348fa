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

#include "kv8_prompt.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kKeys = 64;              // keys of a unit
constexpr int kPanel = kKeys * 128;    // bytes of a [64 keys][64 f16] swizzled image
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

// The word that a wait of a kernel here, having given up, leaves its code in.
__device__ int g_error;

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
      const int row_hi = r >= sr1 ? 0 : a.causal ? min(keys.hi, p + 1) : keys.hi, row_lo = a.window ? p - a.window + 1 : 0;
      // every row of the slot sees the keys [all_lo, all_hi)
      const int all_hi = a.causal ? min(keys.hi, len - T + sr0 / a.group + 1) : keys.hi;
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
        float top = m;
        if (careful)
          top = row_max<true>(k, 0, x[0], top), top = row_max<true>(k, 32, x[1], top);
        else
          top = row_max<false>(k, 0, x[0], top), top = row_max<false>(k, 32, x[1], top);
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
        if (careful)
          l = row_exp<true>(k, 0, x[0], base, l, w[0]), l = row_exp<true>(k, 32, x[1], base, l, w[1]);
        else
          l = row_exp<false>(k, 0, x[0], base, l, w[0]), l = row_exp<false>(k, 32, x[1], base, l, w[1]);
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
      // after a wait that gave up nothing is brought or waited for, but every warp still passes every named barrier
      ok = ok && warp_wait(staged, i & 1, err, kErrTimeoutFull);
      uint2 raw[kSteps];
#pragma unroll
      for (int e = 0; e < kSteps; ++e) raw[e] = lds64(from + e * kStep * D);
      named_barrier(is_v ? 2 : 1, 128);  // the staging tile is read
      if (ok && copies && i + 1 < units) copy(i + 1, id_next);
      if (i >= S::units) ok = ok && warp_wait(&empty[at], ((i / S::units) - 1) & 1, err, kErrTimeoutEmpty);
      if (S::q_smem == 0 && is_v && i == 1) ok = ok && warp_wait(&bar.q_full[0], 0, err, kErrTimeoutEmpty);  // Q has passed
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
  const long long chunk = ((span + want - 1) / want + 127) / 128 * 128;
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
