// C ABI of the 8-bit KV cache: argument checks and dispatch.
#include <atomic>
#include <cmath>
#include <cstdint>

#include "kv8.cuh"

using namespace qhtp;

namespace {

QhtpStatus invalid(const char* msg) {
  set_last_message(msg);
  return QHTP_STATUS_INVALID_ARGUMENT;
}
QhtpStatus unsupported(const char* msg) {
  set_last_message(msg);
  return QHTP_STATUS_UNSUPPORTED;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Shapes only: no pointer is looked at.
QhtpStatus check_shapes(const QhtpKv8Cache& c, const QhtpKv8Seqs& s) {
  if (c.num_blocks <= 0 || c.kv_heads == 0) return invalid("kv8: the cache needs blocks and heads");
  if (c.num_blocks > 0x7fffffffll / c.kv_heads) return unsupported("kv8: at most 2^31 - 1 (block, kv head) tiles");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return unsupported("kv8: head_dim must be 64, 128 or 256");
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return unsupported("kv8: block_size must be 16, 32, 64 or 128");
  if (c.kv_heads > 16383) return unsupported("kv8: at most 16383 kv heads");
  if (s.batch > 65535) return unsupported("kv8: at most 65535 sequences in a call");
  if (s.tokens > (1u << 30)) return unsupported("kv8: at most 2^30 tokens of a sequence in a call");
  if (s.max_blocks > (1u << 30) / c.block_size) return unsupported("kv8: at most 2^30 tokens of context");
  if (s.total < 0) return invalid("kv8: negative total");
  return QHTP_STATUS_OK;
}

QhtpStatus check_pointers(const QhtpKv8Cache& c, const QhtpKv8Seqs& s) {
  if (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr)
    return invalid("kv8: null cache pointer");
  if (!aligned16(c.k) || !aligned16(c.v)) return invalid("kv8: the cache's codes must be 16-byte aligned");
  if (s.block_table == nullptr && s.max_blocks != 0) return invalid("kv8: null block table");
  return QHTP_STATUS_OK;
}

QhtpStatus check_rows(const QhtpKv8Rows& r, int esize) {
  if (r.data == nullptr) return invalid("kv8: null rows");
  const int64_t all = r.batch_stride | r.token_stride | r.head_stride;
  if (!aligned16(r.data) || ((all * esize) & 15) != 0)
    return invalid("kv8: rows must start at, and be apart by, multiples of 16 bytes");
  return QHTP_STATUS_OK;
}

kv8::Pages pages_of(const QhtpKv8Cache& c) {
  int log2 = 4;
  while ((1u << log2) < c.block_size) ++log2;
  return {c.k, c.v, c.k_scale, c.v_scale, c.num_blocks, static_cast<int>(c.kv_heads), log2};
}
kv8::Seqs seqs_of(const QhtpKv8Seqs& s) {
  // no start reaches past 2^31 - 1, and products of total stay in 64 bits
  return {s.block_table,  s.table_stride, static_cast<int>(s.max_blocks), static_cast<int>(s.batch), s.seq_start,
          static_cast<int>(s.tokens), s.total < 0x7fffffff ? s.total : 0x7fffffff};
}
kv8::Rows rows_of(const QhtpKv8Rows& r) { return {r.data, r.batch_stride, r.token_stride, r.head_stride}; }

QhtpStatus check_move(const QhtpKv8Move* m, Kv8Move* out) {
  if (m == nullptr) return invalid("kv8: null argument");
  QhtpStatus st = check_shapes(m->cache, m->seqs);
  if (st != QHTP_STATUS_OK) return st;
  if (m->dtype > QHTP_DTYPE_F32) return unsupported("kv8: rows must be bf16, f16 or f32");
  const bool none = m->seqs.batch == 0 || m->seqs.tokens == 0 || (m->seqs.seq_start != nullptr && m->seqs.total == 0);
  if (none) {
    out->seqs.batch = 0;
    return QHTP_STATUS_OK;
  }
  if ((st = check_pointers(m->cache, m->seqs)) != QHTP_STATUS_OK) return st;
  if (m->first == nullptr) return invalid("kv8: null positions");
  const int esize = m->dtype == QHTP_DTYPE_F32 ? 4 : 2;
  if ((st = check_rows(m->k, esize)) != QHTP_STATUS_OK || (st = check_rows(m->v, esize)) != QHTP_STATUS_OK) return st;
  out->pages = pages_of(m->cache);
  out->seqs = seqs_of(m->seqs);
  out->first = m->first;
  out->k = rows_of(m->k);
  out->v = rows_of(m->v);
  out->dtype = m->dtype;
  out->head_dim = static_cast<int>(m->cache.head_dim);
  out->stream = static_cast<cudaStream_t>(m->stream);
  return QHTP_STATUS_OK;
}

// SMs of the current device, looked up once per device.
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms;
  if (const int n = known[dev].load(std::memory_order_relaxed)) return n;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev].store(sms);
  return sms;
}

// Shapes and plan.  a->seqs.batch is 0 where there is nothing to do.
QhtpStatus plan_attention(const QhtpKv8Attention* run, Kv8Attn* a) {
  if (run == nullptr) return invalid("kv8: null argument");
  QhtpStatus st = check_shapes(run->cache, run->seqs);
  if (st != QHTP_STATUS_OK) return st;
  if (run->dtype != QHTP_DTYPE_BF16 && run->dtype != QHTP_DTYPE_F16) return unsupported("kv8: q must be bf16 or f16");
  if (run->q_heads == 0 || run->q_heads % run->cache.kv_heads != 0)
    return invalid("kv8: q_heads must be a multiple of kv_heads");
  if (!(run->scale > 0.0f) || !std::isfinite(run->scale)) return invalid("kv8: scale must be finite and above 0");
  if (run->window != 0 && !run->causal) return unsupported("kv8: a window needs causal attention");
  if (run->window > (1u << 30)) return unsupported("kv8: window above 2^30");
  a->pages = pages_of(run->cache);
  a->seqs = seqs_of(run->seqs);
  a->head_dim = static_cast<int>(run->cache.head_dim);
  a->q_heads = static_cast<int>(run->q_heads);
  a->group = a->q_heads / a->pages.heads;
  if (static_cast<long long>(a->seqs.tokens) * a->group > (1ll << 30)) return unsupported("kv8: too many rows");
  a->causal = run->causal != 0;
  a->window = static_cast<int>(run->window);
  a->scale_log2 = run->scale * 1.44269504088896341f;
  if (!std::isfinite(a->scale_log2)) return invalid("kv8: scale times log2(e) must be finite");
  a->bf16 = run->dtype == QHTP_DTYPE_BF16;
  const long long cap = static_cast<long long>(run->seqs.max_blocks) * run->cache.block_size;
  a->max_len = static_cast<int>(run->max_len < cap ? run->max_len : cap);
  if (a->seqs.batch == 0 || a->seqs.tokens == 0 || (a->seqs.start != nullptr && a->seqs.total == 0)) {
    a->seqs.batch = 0;
    a->chunks = 1;
    return QHTP_STATUS_OK;
  }
  // Rows of a (sequence, kv head) that one group of the few-row kernel holds stay there; more would read the keys once per group.
  // Measured: 24 rows of head_dim 64 41 us there, 53 on the prompt kernels; 42 rows of head_dim 128 54 and 37, 48 rows 163 and 63;
  // 40 rows of head_dim 256 54 and 32.  (Above 16 rows with keys cut for three CTAs an SM where two fit.)
  a->prompt = static_cast<long long>(a->seqs.tokens) * a->group > (a->head_dim == 256 ? 16 : 32);
  if (a->prompt)
    kv8_prompt_plan(*a, sm_count());
  else
    kv8_decode_plan(*a, sm_count());
  kv8::place_parts(*a);
  if (a->prompt && a->row_groups > 65535) return unsupported("kv8: too many rows");
  if (static_cast<long long>(a->chunks) * a->pages.heads > (1ll << 30)) return unsupported("kv8: too many chunks");
  if (static_cast<long long>(a->pages.heads) * a->row_groups > (1ll << 30)) return unsupported("kv8: too many rows");
  return QHTP_STATUS_OK;
}

// The attention kernels' error words, in the order of qhtp_selftest_kv8_timeout.
constexpr cudaError_t (*kWords[])(int**) = {kv8_decode_word, kv8_prompt_word, kv8_prompt2_word};

}  // namespace

extern "C" {

QhtpStatus qhtp_kv8_write(const QhtpKv8Move* move) {
  Kv8Move m{};
  const QhtpStatus st = check_move(move, &m);
  if (st != QHTP_STATUS_OK || m.seqs.batch == 0) return st;
  return status_from_cuda(launch_kv8_write(m));
}

QhtpStatus qhtp_kv8_read(const QhtpKv8Move* move) {
  Kv8Move m{};
  const QhtpStatus st = check_move(move, &m);
  if (st != QHTP_STATUS_OK || m.seqs.batch == 0) return st;
  return status_from_cuda(launch_kv8_read(m));
}

size_t qhtp_kv8_attention_workspace_bytes(const QhtpKv8Attention* run) {
  Kv8Attn a{};
  return plan_attention(run, &a) == QHTP_STATUS_OK ? kv8_part_bytes(a) : 0;
}

QhtpStatus qhtp_kv8_attention(const QhtpKv8Attention* run) {
  Kv8Attn a{};
  QhtpStatus st = plan_attention(run, &a);
  if (st != QHTP_STATUS_OK || a.seqs.batch == 0) return st;
  if ((st = check_pointers(run->cache, run->seqs)) != QHTP_STATUS_OK) return st;
  if (run->lengths == nullptr) return invalid("kv8: null lengths");
  if ((st = check_rows(run->q, 2)) != QHTP_STATUS_OK || (st = check_rows(run->out, 2)) != QHTP_STATUS_OK) return st;
  const size_t need = kv8_part_bytes(a);
  if (need != 0 && (run->workspace == nullptr || run->workspace_bytes < need || (reinterpret_cast<uintptr_t>(run->workspace) & 255)))
    return invalid("kv8: the workspace is missing, too small or not 256-byte aligned");
  a.lengths = run->lengths;
  a.q = rows_of(run->q);
  a.out = rows_of(run->out);
  a.lse = run->lse;
  a.part = static_cast<float*>(run->workspace);
  a.stream = static_cast<cudaStream_t>(run->stream);
  cudaError_t e = a.prompt ? (a.tile_rows == 256 ? launch_kv8_prompt2(a) : launch_kv8_prompt(a)) : launch_kv8_decode(a);
  if (e == cudaSuccess && (a.chunks > 1 || a.fit)) e = launch_kv8_combine(a);
  return status_from_cuda(e);
}

QhtpStatus qhtp_kv8_check(int* device_code, void* stream) {
  int code = 0;
  for (auto find : kWords) {
    int *word = nullptr, one = 0;
    cudaError_t e = find(&word);
    if (e == cudaSuccess) e = kv8_take_error(word, &one, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return status_from_cuda(e);
    if (code == 0) code = one;
  }
  if (device_code != nullptr) *device_code = code;
  if (code == 0) return QHTP_STATUS_OK;
  set_last_message("kv8: a wait inside an attention kernel gave up");
  return QHTP_STATUS_RUNTIME_ERROR;
}

QhtpStatus qhtp_selftest_kv8_timeout(uint32_t kernel, int* warps_gave_up, uint64_t limit_cycles, void* stream) {
  if (kernel >= sizeof(kWords) / sizeof(kWords[0])) return invalid("kv8: no such kernel");
  if (warps_gave_up == nullptr) return invalid("kv8: null counter");
  int* word = nullptr;
  const cudaError_t e = kWords[kernel](&word);
  if (e != cudaSuccess) return status_from_cuda(e);
  return qhtp_selftest_wait_timeout(word, warps_gave_up, limit_cycles, stream);
}

}  // extern "C"
