// Attention of one new token per sequence over the paged cache, in the prover's integers
// (grape_kv_attend): every row's scores, exp arguments and values, softmax and output, exactly.
//
// The softmax is rounded with the whole row's sum before it meets the values, so nothing can be rescaled
// later: three passes, joined by an integer maximum and integer sums, whose order changes no bit.
#include <algorithm>
#include <exception>

#include "kv.cuh"

namespace grape {

struct AttendArgs {
  KvView c;
  const int32_t *len, *selected;
  uint32_t n_select;
  const int32_t* q;
  uint64_t q_stride;
  uint32_t heads, group, score_shift, soft_shift;
  const int32_t* exp;
  int32_t exp_low;
  uint32_t exp_len;
  uint64_t max_keys;
  int32_t *out, *score, *score_rem, *exp_in, *exp_out, *softmax, *out_rem;
  int64_t* sum;
  int32_t* chunk_max;  // [batch][heads][chunks]
  int64_t* acc;        // [batch][heads][head_dim]
  uint32_t chunks, chunk_keys;
};

// Columns of a row that can hold a position: its length, or the slots of the selected pages.
__device__ __forceinline__ uint32_t columns(const AttendArgs& a, uint32_t b, bool report) {
  const uint32_t n = kv_length(a.c, a.len, b, a.selected ? ~0ull : a.max_keys, report);
  if (!a.selected) return n;
  if (n == 0) return 0;
  const uint64_t all = (uint64_t)a.n_select * a.c.page_size;
  return (uint32_t)min(all, a.max_keys);
}

// Page and slot of column i, or page -1 where the column holds no position.
__device__ __forceinline__ int32_t column_page(const AttendArgs& a, uint32_t b, uint32_t g, uint32_t n, uint32_t i, uint32_t& slot,
                                               bool report) {
  const KvView& c = a.c;
  uint32_t at = c.by_page.div(i);
  slot = i - at * c.page_size;
  if (a.selected) {
    const int32_t s = __ldg(a.selected + ((uint64_t)b * c.kv_heads + g) * a.n_select + at);
    if (s < 0) return -1;
    at = (uint32_t)s;
    if (at >= c.width) {
      if (report) kv_flag(c, STATUS_KV_PLACE);
      return -1;
    }
  }
  if ((uint64_t)at * c.page_size + slot >= n) return -1;
  const int32_t page = kv_page(c, b, at);
  if (page < 0 && report) kv_flag(c, STATUS_KV_PLACE);
  return page;
}

constexpr int AT_THREADS = 256;

// Scores of one head over a chunk of columns, a warp a column; the chunk's largest.
template <int EB>
__global__ void __launch_bounds__(AT_THREADS) k_kv_scores(AttendArgs a) {
  __shared__ int32_t s_max[AT_THREADS / 32];
  const KvView& c = a.c;
  const uint32_t chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, h = row % a.heads, b = row / a.heads, g = h / a.group;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = c.head_dim;
  const uint32_t n = kv_length(c, a.len, b, a.selected ? ~0ull : a.max_keys, false), cols = columns(a, b, chunk == 0 && threadIdx.x == 0);
  if (chunk == 0) {
    for (uint32_t d = threadIdx.x; d < D; d += AT_THREADS) a.acc[(uint64_t)row * D + d] = 0;
    if (threadIdx.x == 0) a.sum[row] = 0;
  }
  const uint32_t first = chunk * a.chunk_keys, last = min(cols, first + a.chunk_keys);
  const int32_t* q = a.q + (uint64_t)b * a.q_stride + (uint64_t)h * D;
  int32_t best = INT32_MIN;
  bool range = false;
  for (uint32_t i = first + warp; i < last; i += AT_THREADS / 32) {
    uint32_t slot;
    const int32_t page = column_page(a, b, g, n, i, slot, lane == 0);
    if (page < 0) continue;
    const char* k = c.k + page * c.page_stride + g * c.head_stride + slot * c.slot_stride;
    int64_t acc = 0;
    for (uint32_t d = lane * 4; d < D; d += 128) {
      const int4 x = __ldg(reinterpret_cast<const int4*>(q + d));
      int4 y;
      if (EB == 4) {
        y = __ldg(reinterpret_cast<const int4*>(k + d * 4));
      } else {
        const short4 s = __ldg(reinterpret_cast<const short4*>(k + d * 2));
        y = make_int4(s.x, s.y, s.z, s.w);
      }
      acc += (int64_t)x.x * y.x + (int64_t)x.y * y.y + (int64_t)x.z * y.z + (int64_t)x.w * y.w;
    }
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(~0u, acc, o);
    const int64_t s = rdiv(acc, a.score_shift);
    const int32_t v = saturate(s, INT32_MIN, INT32_MAX, range);
    best = max(best, v);
    if (lane == 0) {
      const uint64_t at = (uint64_t)row * a.max_keys + i;
      a.score[at] = v;
      if (a.score_rem) a.score_rem[at] = (int32_t)(uint32_t)((uint64_t)acc - ((uint64_t)s << a.score_shift));
    }
  }
  if (range) kv_flag(c, STATUS_KV_RANGE);
  if (lane == 0) s_max[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < AT_THREADS / 32; w++) best = max(best, s_max[w]);
    a.chunk_max[(uint64_t)row * a.chunks + chunk] = best;
  }
}

__global__ void __launch_bounds__(AT_THREADS) k_kv_exp(AttendArgs a) {
  __shared__ int32_t s_max;
  __shared__ unsigned long long s_sum;
  const KvView& c = a.c;
  const uint32_t chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, h = row % a.heads, b = row / a.heads, g = h / a.group;
  const uint32_t n = kv_length(c, a.len, b, a.selected ? ~0ull : a.max_keys, false), cols = columns(a, b, false);
  const uint32_t first = chunk * a.chunk_keys, last = min(cols, first + a.chunk_keys);
  if (first >= last) return;
  if (threadIdx.x == 0) { s_max = INT32_MIN; s_sum = 0; }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.chunks; i += AT_THREADS) atomicMax(&s_max, a.chunk_max[(uint64_t)row * a.chunks + i]);
  __syncthreads();
  const int64_t top = s_max;
  int64_t sum = 0;
  bool outside = false;
  for (uint32_t i = first + threadIdx.x; i < last; i += AT_THREADS) {
    uint32_t slot;
    if (column_page(a, b, g, n, i, slot, false) < 0) continue;
    const uint64_t at = (uint64_t)row * a.max_keys + i;
    int64_t x = a.score[at] - top;
    if (x < a.exp_low) { x = a.exp_low; outside = true; }
    int32_t e = __ldg(a.exp + (x - a.exp_low));
    if (e < 0) { e = 0; outside = true; }
    if (a.exp_in) a.exp_in[at] = (int32_t)x;
    a.exp_out[at] = e;
    sum += e;
  }
  if (outside) kv_flag(c, STATUS_KV_EXP);
  atomicAdd(&s_sum, (unsigned long long)sum);
  __syncthreads();
  if (threadIdx.x == 0) atomicAdd(reinterpret_cast<unsigned long long*>(a.sum + row), s_sum);
}

// Softmax of a chunk and its part of the output, a thread four channels.
template <int EB>
__global__ void __launch_bounds__(AT_THREADS) k_kv_values(AttendArgs a) {
  __shared__ int32_t s_o[AT_THREADS];
  __shared__ int64_t s_at[AT_THREADS];
  const KvView& c = a.c;
  const uint32_t chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, h = row % a.heads, b = row / a.heads, g = h / a.group;
  const uint32_t D = c.head_dim;
  const uint32_t n = kv_length(c, a.len, b, a.selected ? ~0ull : a.max_keys, false), cols = columns(a, b, false);
  const uint32_t first = chunk * a.chunk_keys, last = min(cols, first + a.chunk_keys);
  if (first >= last) return;
  const int64_t sum = a.sum[row];
  for (uint32_t base = first; base < last; base += AT_THREADS) {
    const uint32_t i = base + threadIdx.x;
    uint32_t slot = 0;
    const int32_t page = i < last ? column_page(a, b, g, n, i, slot, false) : -1;
    int32_t o = 0;
    if (page >= 0) {
      const uint64_t at = (uint64_t)row * a.max_keys + i;
      if (sum > 0) o = (int32_t)((((int64_t)a.exp_out[at] << a.soft_shift) + sum / 2) / sum);
      if (a.softmax) a.softmax[at] = o;
    }
    __syncthreads();
    s_o[threadIdx.x] = o;
    s_at[threadIdx.x] = page >= 0 ? page * c.page_stride + g * c.head_stride + slot * c.slot_stride : -1;
    __syncthreads();
    const uint32_t m = min((uint32_t)AT_THREADS, last - base);
    for (uint32_t d = threadIdx.x * 4; d < D; d += AT_THREADS * 4) {
      int64_t acc[4] = {};
      for (uint32_t j = 0; j < m; j++) {
        if (s_at[j] < 0 || s_o[j] == 0) continue;
        int4 y;
        if (EB == 4) {
          y = __ldg(reinterpret_cast<const int4*>(c.v + s_at[j] + d * 4));
        } else {
          const short4 s = __ldg(reinterpret_cast<const short4*>(c.v + s_at[j] + d * 2));
          y = make_int4(s.x, s.y, s.z, s.w);
        }
        const int64_t w = s_o[j];
        acc[0] += w * y.x;
        acc[1] += w * y.y;
        acc[2] += w * y.z;
        acc[3] += w * y.w;
      }
      for (int j = 0; j < 4; j++) atomicAdd(reinterpret_cast<unsigned long long*>(a.acc + (uint64_t)row * D + d + j), (unsigned long long)acc[j]);
    }
  }
}

__global__ void __launch_bounds__(AT_THREADS) k_kv_out(AttendArgs a, uint64_t total) {
  const uint64_t i = (uint64_t)blockIdx.x * AT_THREADS + threadIdx.x;
  if (i >= total) return;
  const uint64_t row = i / a.c.head_dim;
  bool range = false;
  const int64_t acc = a.acc[i], y = rdiv(acc, a.soft_shift);
  a.out[i] = saturate(y, INT32_MIN, INT32_MAX, range);
  if (a.out_rem) a.out_rem[i] = (int32_t)(uint32_t)((uint64_t)acc - ((uint64_t)y << a.soft_shift));
  if (range) kv_flag(a.c, STATUS_KV_RANGE);
  if (i == row * a.c.head_dim && a.sum[row] == 0 && columns(a, (uint32_t)(row / a.heads), false)) kv_flag(a.c, STATUS_KV_EXP);
}

static int attend_launch(grape_ctx* ctx, const grape_kv_cache* cache, AttendArgs& a) {
  const uint64_t rows = (uint64_t)a.c.batch * a.heads, D = cache->head_dim;
  a.chunk_keys = 256;
  const uint64_t all = a.selected ? (uint64_t)a.n_select * cache->page_size : (uint64_t)a.c.width * cache->page_size;
  const uint64_t chunks = (std::min(all, a.max_keys) + a.chunk_keys - 1) / a.chunk_keys;
  if (rows * chunks > 0x7fffffffu || rows * D > (uint64_t(1) << 38))
    return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many rows and columns for one call");
  a.chunks = (uint32_t)chunks;
  auto up = [](uint64_t n) { return (n + 255) & ~uint64_t(255); };
  const uint64_t b_max = up(rows * chunks * 4), b_acc = up(rows * D * 8), b_sum = a.sum ? 0 : up(rows * 8);
  const uint64_t b_keys = up(rows * a.max_keys * 4);
  void* w = nullptr;
  if (int rc = kv_workspace(ctx, b_max + b_acc + b_sum + (a.score ? 0 : b_keys) + (a.exp_out ? 0 : b_keys), &w)) return rc;
  char* p = reinterpret_cast<char*>(w);
  a.chunk_max = reinterpret_cast<int32_t*>(p);
  p += b_max;
  a.acc = reinterpret_cast<int64_t*>(p);
  p += b_acc;
  if (!a.sum) { a.sum = reinterpret_cast<int64_t*>(p); p += b_sum; }
  if (!a.score) { a.score = reinterpret_cast<int32_t*>(p); p += b_keys; }
  if (!a.exp_out) { a.exp_out = reinterpret_cast<int32_t*>(p); p += b_keys; }
  const uint32_t grid = (uint32_t)(rows * chunks);
  if (cache->bits == 32) k_kv_scores<4><<<grid, AT_THREADS, 0, ctx->stream>>>(a);
  else k_kv_scores<2><<<grid, AT_THREADS, 0, ctx->stream>>>(a);
  k_kv_exp<<<grid, AT_THREADS, 0, ctx->stream>>>(a);
  if (cache->bits == 32) k_kv_values<4><<<grid, AT_THREADS, 0, ctx->stream>>>(a);
  else k_kv_values<2><<<grid, AT_THREADS, 0, ctx->stream>>>(a);
  k_kv_out<<<(uint32_t)((rows * D + AT_THREADS - 1) / AT_THREADS), AT_THREADS, 0, ctx->stream>>>(a, rows * D);
  ctx->launches += 4;
  GRAPE_CUDA_TRY(ctx, cudaGetLastError());
  return GRAPE_OK;
}

}  // namespace grape

using namespace grape;

extern "C" int grape_kv_attend(grape_ctx* ctx, const grape_kv_cache* cache, const int32_t* d_table, uint32_t table_width,
                               uint32_t batch, const int32_t* d_len, const int32_t* d_selected, uint32_t n_select,
                               const int32_t* d_q, uint64_t q_stride, uint32_t heads, uint32_t score_shift,
                               const int32_t* d_exp, int32_t exp_low, uint32_t exp_len, uint32_t soft_shift,
                               uint64_t max_keys, int32_t* d_out, const grape_kv_witness* witness) try {
  if (int rc = kv_check_cache(ctx, cache, d_table, table_width, batch, true, true, false)) return rc;
  if (heads < 1 || heads > 65535 || heads % cache->kv_heads)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "heads must be a multiple of kv_heads up to 65535, not %u", heads);
  if (score_shift > 31) return kv_refuse(ctx, GRAPE_ERR_INVALID, "score_shift must be at most 31, not %u", score_shift);
  if (soft_shift < 1 || soft_shift > 20) return kv_refuse(ctx, GRAPE_ERR_INVALID, "soft_shift must be 1 to 20, not %u", soft_shift);
  if (max_keys < 1 || max_keys > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_INVALID, "max_keys must be 1 to 2^31 - 1");
  if (!d_exp || misaligned(d_exp, 4) || exp_low > 0 || (int64_t)exp_low + exp_len < 1)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "the exp table must be given and hold the argument 0");
  if (d_selected ? n_select < 1 || n_select > (1u << 20) : n_select != 0)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "n_select must be 1 to 2^20 with selected pages and 0 without, not %u", n_select);
  if ((uint64_t)n_select * cache->page_size > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "n_select * page_size must stay below 2^31");
  const grape_kv_witness none = {};
  const grape_kv_witness& w = witness ? *witness : none;
  if (batch) {
    if (int rc = kv_check_rows(ctx, "queries", d_q, q_stride, (uint64_t)heads * cache->head_dim)) return rc;
    if (!d_len || misaligned(d_len, 4)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "lengths must be given, on 4 bytes");
    if (!d_out) return kv_refuse(ctx, GRAPE_ERR_INVALID, "no output");
  }
  if (misaligned(d_selected, 4) || misaligned(d_out, 16) || misaligned(w.d_out_rem, 16) || misaligned(w.d_score, 16) || misaligned(w.d_score_rem, 16) ||
      misaligned(w.d_exp_in, 16) || misaligned(w.d_exp_out, 16) || misaligned(w.d_softmax, 16) || misaligned(w.d_sum, 8))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "outputs must be on 16 bytes");
  if ((uint64_t)batch * heads > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many sequences and heads for one call");
  if (!ctx) return kv_refuse(ctx, GRAPE_ERR_INVALID, "null context");
  make_device_current(ctx);
  if (!batch) return GRAPE_OK;
  AttendArgs a{};
  a.c = kv_view(ctx, cache, d_table, table_width, batch);
  a.len = d_len;
  a.selected = d_selected;
  a.n_select = n_select;
  a.q = d_q;
  a.q_stride = q_stride;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.score_shift = score_shift;
  a.soft_shift = soft_shift;
  a.exp = d_exp;
  a.exp_low = exp_low;
  a.exp_len = exp_len;
  a.max_keys = max_keys;
  a.out = d_out;
  a.score = w.d_score;
  a.score_rem = w.d_score_rem;
  a.exp_in = w.d_exp_in;
  a.exp_out = w.d_exp_out;
  a.softmax = w.d_softmax;
  a.sum = w.d_sum;
  a.out_rem = w.d_out_rem;
  return attend_launch(ctx, cache, a);
} catch (const std::exception& e) {
  return kv_refuse(nullptr, GRAPE_ERR_NOMEM, "%s", e.what());
}
