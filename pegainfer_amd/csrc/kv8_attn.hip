// Softmax attention over the 8-bit paged cache, and the weight that every cached token gets.
//
//   o[r, h] = sum_j p_j v_j,  p = softmax_j(scale q[r, h] . k_j) over the slots j <= starts[e] + i of row i of entry e
//   mass_out[j, g] = keep mass[j, g] + sum over the entry's rows r and the query heads h of kv head g of p_j[r, h]
#include <algorithm>

#include "kv8_host.h"

namespace pk {

__device__ __forceinline__ f32x4 mfma16(const bf16x8_t& a, const bf16x8_t& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// over the four lanes that hold a row's scores
__device__ __forceinline__ float quad_max(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float quad_sum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }

struct AttnArgs {
  Kv8 c;
  const void* q;
  int64_t q_stride, out_stride;
  const int32_t *row0, *starts;
  int n_rows, group, heads;
  float scale_log2;
  void* out;
  float* lse;            // [n_rows][heads], log2 of the sum of exp(scores); NULL: not wanted
};

// the queries' rows of a kv head, (token, head of the group) in order; row n of a tile of sixteen is the lane's
struct QueryRow { int row, head, far; };   // far: the last slot that it sees; -1: no such row
__device__ __forceinline__ QueryRow query_row(int rr, int total, int group, const RowSpan& rows, int start, int kv_head) {
  if (rr >= total) return {rows.first, kv_head * group, -1};
  const int tok = rr / group;
  return {rows.first + tok, kv_head * group + rr - tok * group, start + tok};
}

// One workgroup of four waves: sixteen query rows of a kv head, the blocks of keys in pairs dealt to the waves, whose states meet in shared memory at the end.
// Scores are computed transposed (keys x rows), so that a lane holds four keys' scores of one row: exactly what the second product wants from it.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void kv8_attn_kernel(AttnArgs a) {
  constexpr int NP = kv8_parts<T>(), C = D / 64;
  __shared__ f32x4 s_o[2][D / 16][64];
  __shared__ float s_m[2][16], s_l[2][16];
  const int e = blockIdx.z, head = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (start < 0 || start > INT32_MAX - 32 - rows.n) return;
  const int len = start + rows.n;
  for (int tile = blockIdx.x; tile * 16 < total; tile += gridDim.x) {
    const QueryRow r = query_row(tile * 16 + n, total, a.group, rows, start, head);
    bf16x8_t qf[C][2][NP];
    const T* qp = static_cast<const T*>(a.q) + r.row * a.q_stride + (int64_t)r.head * D + g * 16;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      kv8_query(qp + c * 64, qf[c][0]);
      kv8_query(qp + c * 64 + 8, qf[c][1]);
    }
    const int last = min(tile * 16 + 15, total - 1) / a.group + start;   // the last slot that any row of the tile sees
    const int blocks = last / kKv8Page + 1;
    float m = -INFINITY, l = 0.f;
    f32x4 o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int b = 2 * wave; b < blocks; b += 8) {
      f32x4 s[2];
      int page[2];
      float vs[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        page[h] = b + h < blocks ? a.c.page(e, b + h) : -1;
        s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
        vs[h] = 0.f;
        if (page[h] >= 0) {
          const uint8_t* kb = a.c.block(page[h], 0, head, D) + n * 64 + g * 16;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(kb + c * 1024);
            const bf16x8_t k0 = kv8_operand<FMT>(w.x, w.y), k1 = kv8_operand<FMT>(w.z, w.w);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) {
              s[h] = mfma16(k0, qf[c][0][p], s[h]);
              s[h] = mfma16(k1, qf[c][1][p], s[h]);
            }
          }
          const float ks = *a.c.scale(page[h], 0, head) * a.scale_log2;
          vs[h] = *a.c.scale(page[h], 1, head);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][i] = (b + h) * kKv8Page + 4 * g + i <= r.far ? s[h][i] * ks : -INFINITY;
        } else {
          s[h] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        }
      }
      float mx = m;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[h][i]);
      mx = quad_max(mx);
      const float base = mx == -INFINITY ? 0.f : mx, alpha = exp2_of(m - base);
      m = mx;
      l *= alpha;
      float p[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[4 * h + i] = exp2_of(s[h][i] - base);
          l += p[4 * h + i];
          p[4 * h + i] *= vs[h];
        }
      bf16x8_t pf[NP];
      kv8_split<NP>(p, pf);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i] *= alpha;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u32x4 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[h] = u32x4{0, 0, 0, 0};
          if (page[h] >= 0) w[h] = *reinterpret_cast<const u32x4*>(a.c.block(page[h], 1, head, D) + c * 1024 + g * 256 + n * 16);
          // what lies behind the entry's last token may be any bytes, and 0 times one of them a NaN
          const int there = len - ((b + h) * kKv8Page + 4 * g);
          if (there < 4) w[h] &= there <= 0 ? 0u : 0xFFFFFFFFu >> (32 - 8 * there);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8_t vf = kv8_operand<FMT>(w[0][j], w[1][j]);
#pragma unroll
          for (int k = NP - 1; k >= 0; --k) o[4 * c + j] = mfma16(vf, pf[k], o[4 * c + j]);
        }
      }
    }
    l = quad_sum(l);
    // four states into one: waves 2, 3 into 0, 1, then 1 into 0
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) s_o[wave - half][i][lane] = o[i];
        if (g == 0) { s_m[wave - half][n] = m; s_l[wave - half][n] = l; }
      }
      __syncthreads();
      if (wave < half) {
        const float mo = s_m[wave][n], both = fmaxf(m, mo), base = both == -INFINITY ? 0.f : both;
        const float x = exp2_of(m - base), y = exp2_of(mo - base);
        m = both;
        l = l * x + s_l[wave][n] * y;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] = o[i] * x + s_o[wave][i][lane] * y;
      }
    }
    if (wave == 0 && r.far >= 0) {
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // no key: zeros
      T* op = static_cast<T*>(a.out) + r.row * a.out_stride + (int64_t)r.head * D + g * 16;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * i + j] = o[4 * c + j][i] * inv;
        Vec8<T>::store(op + c * 64, x);
        Vec8<T>::store(op + c * 64 + 8, x + 8);
      }
      if (a.lse && g == 0) a.lse[(int64_t)r.row * a.heads + r.head] = l > 0.f || l != l ? m + __log2f(l) : INFINITY;
    }
    __syncthreads();
  }
}

// The weights that a step gives to the cached tokens, from the sums that the attention left: a wave a block of keys, which it holds as operands while it walks
// all rows that see them, so that every token's sum is one wave's, in the rows' order.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void kv8_mass_kernel(AttnArgs a, const float* mass, int64_t mass_stride, float* out, int64_t out_stride, float keep) {
  constexpr int NP = kv8_parts<T>(), C = D / 64;
  const int e = blockIdx.z, head = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 32 - rows.n) return;
  const int len = start + rows.n;
  for (int b = blockIdx.x * 4 + wave; b * kKv8Page < len; b += gridDim.x * 4) {
    const int page = a.c.page(e, b);
    if (page < 0) continue;
    bf16x8_t kf[C][2];
    const uint8_t* kb = a.c.block(page, 0, head, D) + n * 64 + g * 16;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(kb + c * 1024);
      kf[c][0] = kv8_operand<FMT>(w.x, w.y);
      kf[c][1] = kv8_operand<FMT>(w.z, w.w);
    }
    const float ks = *a.c.scale(page, 0, head) * a.scale_log2;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int first = max(b * kKv8Page - start, 0) * a.group / 16;     // the first tile with a row that sees the block
    for (int tile = first; tile * 16 < total; ++tile) {
      const QueryRow r = query_row(tile * 16 + n, total, a.group, rows, start, head);
      const T* qp = static_cast<const T*>(a.q) + r.row * a.q_stride + (int64_t)r.head * D + g * 16;
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        bf16x8_t q0[NP], q1[NP];
        kv8_query(qp + c * 64, q0);
        kv8_query(qp + c * 64 + 8, q1);
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {
          s = mfma16(kf[c][0], q0[p], s);
          s = mfma16(kf[c][1], q1[p], s);
        }
      }
      const float lse = a.lse[(int64_t)r.row * a.heads + r.head];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += b * kKv8Page + 4 * g + i <= r.far ? exp2_of(s[i] * ks - lse) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = row16_sum(sum[i]);
      const int t = 4 * g + i;
      if (n == i && b * kKv8Page + t < len) {
        const int64_t at = head * kKv8Page + t;
        // 0 means without what was there, whatever that is
        out[page * out_stride + at] = keep == 0.f ? x : fmaf(keep, mass[page * mass_stride + at], x);
      }
    }
  }
}

}  // namespace pk

using namespace pk;

extern "C" {

int64_t pegainfer_kv8_attention_workspace(int32_t n_rows, int32_t heads, int32_t with_mass) {
  return with_mass ? (int64_t)std::max(n_rows, 0) * std::max(heads, 0) : 0;
}

pegainfer_status_t pegainfer_kv8_attention(const pegainfer_kv8_cache* cache, const pegainfer_kv8_attn_desc* d, pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || !d || (d->dtype != kDtBf16 && d->dtype != kDtF32) || d->heads < 1 || d->heads % cache->kv_heads || d->n_rows < 0 || d->max_rows < 0 || d->max_len < 0)
    return PK_BAD;
  if (d->n_rows == 0 || d->max_rows == 0 || cache->n_entries == 0) return 0;
  const int64_t width = (int64_t)d->heads * cache->dim, unit = d->dtype == kDtBf16 ? 8 : 4;
  if (!d->q || !d->out || !d->row0 || !d->starts || !host_aligned16(d->q) || !host_aligned16(d->out) || d->q_row_stride < width || d->out_row_stride < width ||
      d->q_row_stride % unit || d->out_row_stride % unit || (int64_t)d->n_rows * (d->heads / cache->kv_heads) > INT32_MAX - 1024)
    return PK_BAD;
  const bool weigh = d->mass_out != nullptr;
  const int64_t mass_width = (int64_t)cache->kv_heads * kKv8Page;
  if (weigh && (d->mass_out_page_stride < mass_width || (d->mass_keep != 0.f && (!d->mass || d->mass_page_stride < mass_width)))) return PK_BAD;
  if (pegainfer_kv8_attention_workspace(d->n_rows, d->heads, weigh) > 0 && !d->workspace) return PK_BAD;
  const Kv8 c = kv8_of(cache);
  const int group = d->heads / cache->kv_heads;
  const AttnArgs a{c, d->q, d->q_row_stride, d->out_row_stride, d->row0, d->starts, d->n_rows, group, d->heads, d->scale * 1.4426950408889634f, d->out,
                   weigh ? d->workspace : nullptr};
  const int rows = std::min(d->max_rows, d->n_rows);
  const dim3 grid(ceil_div((int64_t)rows * group, 16), c.kv_heads, c.entries);
  const dim3 mass_grid(std::max(1, ceil_div(d->max_len, 4 * kKv8Page)), c.kv_heads, c.entries);
  kv8_by(d->dtype, cache->format, cache->dim, [&](auto* t, auto fmt, auto dim) {
    using T = std::remove_pointer_t<decltype(t)>;
    kv8_attn_kernel<T, fmt(), dim()><<<grid, 256, 0, as_stream(stream)>>>(a);
    if (weigh)
      kv8_mass_kernel<T, fmt(), dim()><<<mass_grid, 256, 0, as_stream(stream)>>>(a, d->mass, d->mass_page_stride, d->mass_out, d->mass_out_page_stride, d->mass_keep);
  });
  return (pegainfer_status_t)hipGetLastError();
}

}  // extern "C"
