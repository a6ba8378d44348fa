// Writing K and V rows into the 8-bit paged cache, and reading them back.
//
// A (block, kv head) tile of the cache has one float32 scale.  Per touched tile, with X the new rows
// that fall into it (all arithmetic float32, every operation correctly rounded):
//
//   s_new = max|X| / 127, 0 below 2^-64, NaN if X holds a NaN or an infinity
//   s     = s_new where the tile's slot 0 is written (the tile starts anew), else max(s_old, s_new) with an s_old
//           below 2^-64 as 0, NaN if either is not finite
//   new codes = clamp(rint(x * (1 / s)), -127, 127), 0 where s is 0 or NaN
//   old codes = rint(c * (s_old / s)) where s grew
//
// One CTA owns one tile of K or of V, so a tile's scale, its old codes and its new ones are read and
// written by that CTA alone: no atomics, and the same bytes in every run.
//
// Per element the input is read once (2 or 4 bytes) and one code byte is written; a
// tile's rows stay in registers between the maximum and the rounding.  Conversions between integers and floats run at a
// quarter of the rate of additions and took longer than the memory here, so both directions go through additions:
// y + 1.5 2^23 leaves rint(y) in its low bits, and 2^23 + (code + 128) is made by placing a byte (20446 tokens of 8 heads
// x 128 written and read back: 93 us with conversions, 76 without).
//
// Measured, 8 heads x 128, blocks of 64: 20446 f16 tokens of 8 sequences written in 29 us (4.3 TB/s; 20480 in 8 equal ones 27, of
// f32 44 us, 4.7 TB/s), read as f32 in 41 us (5.1 TB/s); 80000 tokens read as bf16 in 83 us (5.9 TB/s).  A write keeps neither
// memory nor issue slots (66 %) busy throughout: each small CTA loads, waits, and stores.  One token of each of 64 sequences is written in 4.5 us, which is the
// chain of a CTA's loads (position, table, old scale and row, old codes where the scale grew), not their bytes.
// Persistent CTAs that fetch the next tile's rows ahead were slower (107 us against 93): the many small CTAs that an SM holds
// overlap better.
#include <type_traits>

#include "kv8.cuh"

namespace qhtp {
namespace kv8 {
namespace {

constexpr int kMaxThreads = 256;

struct MoveArgs {
  Pages pages;
  Seqs seqs;
  const int32_t* first;
  Rows row[2];   // K, V
  int vec_log2;  // 16-byte vectors of a row
};

// rint of two's-complement bytes: the low byte of y + 1.5 2^23, |y| < 2^22 (y here is at most 127 and a rounding).
__device__ __forceinline__ uint32_t round_bits(float y) { return __float_as_uint(__fadd_rn(y, 12582912.0f)); }
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return prmt(prmt(a, b, 0x0040u), prmt(c, d, 0x0040u), 0x5410u);
}
// Four int8 codes -> float32, exactly.
__device__ __forceinline__ void codes_to_float(uint32_t w, float (&f)[4]) {
  w ^= 0x80808080u;
  f[0] = __uint_as_float(prmt(w, 0x4b000000u, 0x7440u)) - 8388736.0f;
  f[1] = __uint_as_float(prmt(w, 0x4b000000u, 0x7441u)) - 8388736.0f;
  f[2] = __uint_as_float(prmt(w, 0x4b000000u, 0x7442u)) - 8388736.0f;
  f[3] = __uint_as_float(prmt(w, 0x4b000000u, 0x7443u)) - 8388736.0f;
}
// The largest |x| of 16 bytes of T, as the bits of T (for the 16-bit types of both halves of the word): magnitudes are
// ordered like their bits, infinity and NaN above all others.
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t top, const uint4& r) {
  if constexpr (Vec<T>::n == 4)
    return max(max(max(top, r.x & 0x7fffffffu), r.y & 0x7fffffffu), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
  else
    return __vmaxu2(__vmaxu2(__vmaxu2(top, r.x & 0x7fff7fffu), r.y & 0x7fff7fffu),
                    __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
}
template <typename T>
__device__ __forceinline__ float max_value(uint32_t top) {
  if constexpr (Vec<T>::n == 4) return __uint_as_float(top);
  top = max(top & 0xffffu, top >> 16);
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(top)));
  return __uint_as_float(top << 16);
}

// One CTA per (block of the sequence, K or V of a head, sequence).  NV: vectors a thread keeps in
// registers; tiles with more than NV per thread read their rows a second time (from L2).
template <typename T, int NV>
__global__ void __launch_bounds__(kMaxThreads, NV <= 4 ? 6 : 3) kv8_write_kernel(const MoveArgs a) {
  constexpr int VN = Vec<T>::n;
  const int b = blockIdx.z, h = blockIdx.y >> 1, kv = blockIdx.y & 1;
  long long row0;
  const int n = seq_rows(a.seqs, b, row0);
  const long long past = max(a.first[b], 0);
  const int bs_log2 = a.pages.bs_log2, bs = 1 << bs_log2;
  const long long blk = (past >> bs_log2) + blockIdx.x;
  const long long lo = max(past, blk << bs_log2), hi = min(past + n, (blk + 1) << bs_log2);
  if (lo >= hi) return;
  const long long id = block_of(a.seqs, a.pages, b, blk);
  if (id < 0) return;
  const int slot0 = static_cast<int>(lo - (blk << bs_log2)), rows = static_cast<int>(hi - lo);

  const Rows& src = a.row[kv];
  const T* x = static_cast<const T*>(src.data) + b * src.batch_stride + (row0 + lo - past) * src.token_stride +
               h * src.head_stride;
  const long long tile = id * a.pages.heads + h;
  const int d = VN << a.vec_log2;
  int8_t* codes = (kv ? a.pages.v : a.pages.k) + tile * bs * d;
  float* scale_at = (kv ? a.pages.v_scale : a.pages.k_scale) + tile;
  // Below kScaleMin it counts as 0: new rows of that size would else be divided by a scale that they may be far above, or
  // by one whose reciprocal is infinite.
  float old = slot0 ? *scale_at : 0.0f;
  if (old < kScaleMin) old = 0.0f;  // a NaN stays

  const int nvec = rows << a.vec_log2, cmask = (1 << a.vec_log2) - 1;
  auto load = [&](int i) {
    return __ldg(reinterpret_cast<const uint4*>(x + (i >> a.vec_log2) * src.token_stride + (i & cmask) * VN));
  };
  uint4 raw[NV];
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * blockDim.x;
    raw[i] = at < nvec ? load(at) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) bits = max_bits<T>(bits, raw[i]);
  for (int at = threadIdx.x + NV * blockDim.x; at < nvec; at += blockDim.x) bits = max_bits<T>(bits, load(at));
  uint32_t top = __float_as_uint(max_value<T>(bits));

  __shared__ uint32_t s_top[kMaxThreads / 32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();  // also: every thread has read the old scale
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) top = max(top, s_top[w]);

  float s = __fdiv_rn(__uint_as_float(top), 127.0f);
  if (s < kScaleMin) s = 0.0f;
  if (slot0) s = fmaxf(s, old);  // fmaxf drops a NaN: both are looked at below
  const bool fine = top < 0x7f800000u && isfinite(old);
  if (!fine) s = nan_f32();
  if (threadIdx.x == 0) *scale_at = s;
  const float inv = fine && s > 0.0f ? __frcp_rn(s) : 0.0f;

  auto put = [&](int at, const uint4& r) {
    float f[VN];
    Vec<T>::load(r, f);
    uint32_t w[VN / 4];
    // s is 0, or at least the rows' own max|x| / 127: no code is above 127
#pragma unroll
    for (int e = 0; e < VN / 4; ++e) {
      const uint32_t c = low_bytes(round_bits(__fmul_rn(f[4 * e], inv)), round_bits(__fmul_rn(f[4 * e + 1], inv)),
                                   round_bits(__fmul_rn(f[4 * e + 2], inv)), round_bits(__fmul_rn(f[4 * e + 3], inv)));
      w[e] = fine ? c : 0u;
    }
    int8_t* to = codes + ((slot0 << a.vec_log2) + at) * VN;
    if constexpr (VN == 8)
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(to) = w[0];
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * blockDim.x;
    if (at < nvec) put(at, raw[i]);
  }
  for (int at = threadIdx.x + NV * blockDim.x; at < nvec; at += blockDim.x) put(at, load(at));

  if (slot0 == 0 || !fine || s == old) return;
  // the scale grew: what the tile held before, in the new scale
  const float ratio = __fdiv_rn(old, s);
  const int words = slot0 * d / 16;
  uint4* held = reinterpret_cast<uint4*>(codes);
  for (int i = threadIdx.x; i < words; i += blockDim.x) {
    const uint4 r = held[i];
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f[4];
      codes_to_float(w[e], f);
      w[e] = low_bytes(round_bits(__fmul_rn(f[0], ratio)), round_bits(__fmul_rn(f[1], ratio)),
                       round_bits(__fmul_rn(f[2], ratio)), round_bits(__fmul_rn(f[3], ratio)));
    }
    held[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Codes that a reading thread takes at a time: 16 for 16-bit rows (two 16-byte stores, a whole sector), 4 for float32.
template <typename T>
constexpr int codes_of() {
  return Vec<T>::n == 8 ? 16 : 4;
}

// One CTA per (block of the sequence, K or V of a head, sequence).
// Rows whose block the table does not map come back as NaN.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads) kv8_read_kernel(const MoveArgs a) {
  constexpr int VN = Vec<T>::n, kCodes = codes_of<T>();
  const int b = blockIdx.z, h = blockIdx.y >> 1, kv = blockIdx.y & 1;
  long long row0;
  const int n = seq_rows(a.seqs, b, row0);
  const long long past = a.first[b];
  const int bs_log2 = a.pages.bs_log2;
  const long long blk = (past >> bs_log2) + blockIdx.x;
  const long long lo = max(past, blk << bs_log2), hi = min(past + n, (blk + 1) << bs_log2);
  if (lo >= hi) return;
  const long long id = block_of(a.seqs, a.pages, b, blk);
  const int slot0 = static_cast<int>(lo - (blk << bs_log2)), rows = static_cast<int>(hi - lo);
  const int d = kCodes << a.vec_log2;
  const long long tile = max(id, 0ll) * a.pages.heads + h;
  const int8_t* codes = (kv ? a.pages.v : a.pages.k) + ((tile << bs_log2) + slot0) * d;
  const float s = id < 0 ? nan_f32() : (kv ? a.pages.v_scale : a.pages.k_scale)[tile];
  const Rows& dst = a.row[kv];
  T* x = static_cast<T*>(dst.data) + b * dst.batch_stride + (row0 + lo - past) * dst.token_stride + h * dst.head_stride;
  const int nvec = rows << a.vec_log2, cmask = (1 << a.vec_log2) - 1;
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    uint32_t w[kCodes / 4];
    if constexpr (kCodes == 16) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(codes) + i);
      w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(codes) + i);
    }
    T* const to = x + (i >> a.vec_log2) * dst.token_stride + (i & cmask) * kCodes;
#pragma unroll
    for (int e = 0; e < kCodes / VN; ++e) {
      float f[VN];
#pragma unroll
      for (int j = 0; j < VN / 4; ++j) {
        float g[4];
        codes_to_float(w[e * VN / 4 + j], g);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[4 * j + k] = __fmul_rn(g[k], s);
      }
      *reinterpret_cast<uint4*>(to + e * VN) = Vec<T>::store(f);
    }
  }
}

// Blocks that the rows of one sequence can touch.
unsigned blocks_touched(const Kv8Move& m) {
  const long long bs = 1ll << m.pages.bs_log2;
  return static_cast<unsigned>((m.seqs.tokens + bs - 2) / bs + 1);
}

int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

template <typename T>
cudaError_t write(const Kv8Move& m) {
  MoveArgs a{m.pages, m.seqs, m.first, {m.k, m.v}, log2_of(m.head_dim / Vec<T>::n)};
  const dim3 grid(blocks_touched(m), 2 * m.pages.heads, m.seqs.batch);
  const int rows = m.seqs.tokens < (1 << m.pages.bs_log2) ? m.seqs.tokens : 1 << m.pages.bs_log2;
  const int vecs = rows * m.head_dim / Vec<T>::n;
  // four vectors a thread where the tile has them: enough loads in flight per thread, and 128 threads
  // at the least, for the tiles of single tokens whose old codes have to be scaled anew
  const int threads = vecs >= 4 * 256 ? 256 : 128;
  const int per = (vecs + threads - 1) / threads;
  if (per <= 1)
    kv8_write_kernel<T, 1><<<grid, threads, 0, m.stream>>>(a);
  else if (per <= 4)
    kv8_write_kernel<T, 4><<<grid, threads, 0, m.stream>>>(a);
  else
    kv8_write_kernel<T, 8><<<grid, threads, 0, m.stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t read(const Kv8Move& m) {
  constexpr int kCodes = codes_of<T>();
  MoveArgs a{m.pages, m.seqs, m.first, {m.k, m.v}, log2_of(m.head_dim / kCodes)};
  const dim3 grid(blocks_touched(m), 2 * m.pages.heads, m.seqs.batch);
  const int rows = m.seqs.tokens < (1 << m.pages.bs_log2) ? m.seqs.tokens : 1 << m.pages.bs_log2;
  const int vecs = rows * m.head_dim / kCodes;
  kv8_read_kernel<T><<<grid, vecs >= 512 ? 256 : 128, 0, m.stream>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace kv8

cudaError_t launch_kv8_write(const Kv8Move& m) {
  if (m.dtype == QHTP_DTYPE_BF16) return kv8::write<__nv_bfloat16>(m);
  if (m.dtype == QHTP_DTYPE_F16) return kv8::write<__half>(m);
  return kv8::write<float>(m);
}

cudaError_t launch_kv8_read(const Kv8Move& m) {
  if (m.dtype == QHTP_DTYPE_BF16) return kv8::read<__nv_bfloat16>(m);
  if (m.dtype == QHTP_DTYPE_F16) return kv8::read<__half>(m);
  return kv8::read<float>(m);
}

}  // namespace qhtp
