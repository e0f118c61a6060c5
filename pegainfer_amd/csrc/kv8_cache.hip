// The 8-bit paged cache's movers: rows in (append), rows out (read), tokens to fresh pages by what they weigh (evict).
// All of them move bytes; a wave owns a block's keys, another its values, and keeps them in registers from load to store.
#include <algorithm>

#include "kv8_host.h"

namespace pk {

// Rows pass the caches by, in and out: they are used once here (prompts written and read back 61 -> 54 us, 62 000 tokens read in fp32 158 -> 151).
// N = 4 or 8 values of a row at 8 or 16 bytes (fp32: 16)
template <int N, typename T>
__device__ __forceinline__ void rows_in(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + i));
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
    typedef __attribute__((ext_vector_type(N / 2))) uint32_t Words;
    const Words v = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[2 * i] = bf_lo(v[i]);
      x[2 * i + 1] = bf_hi(v[i]);
    }
  }
}
// 16 bytes of a row
__device__ __forceinline__ void rows_out(float* p, const float* x) { __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4*>(p)); }
__device__ __forceinline__ void rows_out(uint16_t* p, const float* x) {
  __builtin_nontemporal_store(u32x4{pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7])}, reinterpret_cast<u32x4*>(p));
}

// ---- where a lane's 16 bytes of a block come from ----
// keys: value c * 64 + 16 q .. + 15 of token n;  values: tokens 4 q .. + 3 of the values 64 c + 4 n .. + 3, byte 4 j + t = value j, token t
__device__ __forceinline__ int unit_at(int side, int chunk, int n, int q) { return chunk * 1024 + (side == 0 ? n * 64 + q * 16 : q * 256 + n * 16); }

// x[16] of a unit from rows of T: row(t) is the row of the block's token t, or -1: zeros.  Such a row's place is read from row `any` and left out, so that no load
// waits behind a branch.
template <typename T, typename Row>
__device__ __forceinline__ void unit_rows(const T* base, int64_t stride, int side, int chunk, int n, int q, Row row, int any, float* x) {
  if (side == 0) {
    const int r = row(n);
    const T* p = base + (r < 0 ? any : r) * stride + chunk * 64 + q * 16;
    rows_in<8>(p, x);
    rows_in<8>(p + 8, x + 8);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = r < 0 ? 0.f : x[i];
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int r = row(4 * q + t);
      float y[4];
      rows_in<4>(base + (r < 0 ? any : r) * stride + chunk * 64 + 4 * n, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * j + t] = r < 0 ? 0.f : y[j];
    }
  }
}
// token (of 16) that value i of a unit belongs to
__device__ __forceinline__ int unit_token(int side, int n, int q, int i) { return side == 0 ? n : 4 * q + (i & 3); }

// Rows into the cache.  One workgroup of two waves a (block, head): the rows' largest value, the exponent it wants (not below that of the tokens in front of
// them in the block), their codes, and the older tokens' codes again where the exponent grew.  Bound by bytes: the rows are read once
// (20 000 tokens of 8 x 128 from bf16: 36 us, 3.4 TB/s; 23 600 from fp32 60, 4.1; 16 single tokens 5 us, a launch).  mass: given, the tokens that the rows bring weigh nothing yet, and the
// slots behind them neither, whatever a page's last owner left there.
// Waves of a SIMD that the registers hold (prompts of up to 8000 rows of 8 x 128 in int8, with what is read back: 53 us with seven, 57 with five)
template <int D> constexpr int append_waves() { return D == 64 ? 8 : D == 128 ? 6 : 4; }
template <typename T, int FMT, int D>
__global__ __launch_bounds__(128, append_waves<D>()) void kv8_append_kernel(Kv8 c, float* mass, int64_t mass_stride, const T* k, const T* v, int64_t k_stride, int64_t v_stride,
                                                         const int32_t* row0, const int32_t* starts, int n_rows) {
  const int e = blockIdx.z, head = blockIdx.y, side = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const RowSpan rows = row_span(row0, e, n_rows);
  const int64_t start = starts[e];
  if (rows.n == 0 || start < 0 || start + rows.n > INT32_MAX - 32) return;
  const T* base = (side == 0 ? k : v) + head * D;
  const int64_t stride = side == 0 ? k_stride : v_stride;
  const int end = (int)start + rows.n;
  for (int b = (int)start / kKv8Page + blockIdx.x, past = (end + kKv8Page - 1) / kKv8Page; b < past; b += gridDim.x) {   // in blocks: slots pass 2^31 a grid behind the last
    const int page = c.page(e, b);
    if (page < 0) continue;
    const int low = b * kKv8Page, first = max((int)start - low, 0);   // tokens 0 .. first - 1 of the block were there before
    if (mass && side == 0 && q == 0 && n >= first) mass[page * mass_stride + head * kKv8Page + n] = 0.f;
    auto row = [&](int t) { const int s = low + t; return s >= start && s < end ? rows.first + (s - (int)start) : -1; };
    float x[D / 64][16], amax = 0.f;
#pragma unroll
    for (int ch = 0; ch < D / 64; ++ch) unit_rows(base, stride, side, ch, n, q, row, rows.first, x[ch]);
#pragma unroll
    for (int ch = 0; ch < D / 64; ++ch) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = fabsf(x[ch][i]);
        amax = a <= 3.4028234e38f ? fmaxf(amax, a) : amax;            // finite values alone say how large the block is
      }
    }
    int ex = kv8_exp<FMT>(fminf(wave_max(amax), kv8_largest<FMT>()));
    uint8_t* blk = c.block(page, side, head, D);
    float* scale = c.scale(page, side, head);
    const int was = first > 0 ? exp_of(*scale) : ex;
    ex = max(ex, was);
    const float to = pow2f(-ex), again = pow2f(was - ex), top = FMT == kE4m3 && ex == 120 ? 240.f : kv8_top<FMT>();      // int8's exponent does not reach 122
#pragma unroll
    for (int ch = 0; ch < D / 64; ++ch) {
      uint8_t* at = blk + unit_at(side, ch, n, q);
      u32x4 old = {0, 0, 0, 0};
      if (first > 0) old = *reinterpret_cast<const u32x4*>(at);
      u32x4 out;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float y[4];
        if (first > 0) kv8_numbers<FMT>(old[w], y);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = first > 0 && unit_token(side, n, q, 4 * w + i) < first ? y[i] * again : x[ch][4 * w + i] * to;
        out[w] = kv8_codes<FMT>(y, top);
      }
      *reinterpret_cast<u32x4*>(at) = out;
    }
    if (lane == 0) *scale = pow2f(ex);
  }
}

// Tokens out of the cache: code * scale, exact in either type.  Bound by bytes, most of them written (62 000 tokens of 8 x 128 to fp32: 151 us, 4.1 TB/s).  Lanes are laid
// over the rows that leave, not over the blocks, so that whole lines do.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(128) void kv8_read_kernel(Kv8 c, T* k, T* v, const int32_t* row0, const int32_t* starts, int n_rows) {
  const int e = blockIdx.z, head = blockIdx.y, side = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const RowSpan rows = row_span(row0, e, n_rows);
  const int64_t start = starts[e];
  if (rows.n == 0 || start < 0 || start + rows.n > INT32_MAX - 32) return;
  const int64_t stride = (int64_t)c.kv_heads * D;
  T* base = (side == 0 ? k : v) + head * D;
  const int end = (int)start + rows.n;
  for (int b = (int)start / kKv8Page + blockIdx.x, past = (end + kKv8Page - 1) / kKv8Page; b < past; b += gridDim.x) {   // in blocks: slots pass 2^31 a grid behind the last
    const int page = c.page(e, b), low = b * kKv8Page;
    const float scale = page < 0 ? 0.f : *c.scale(page, side, head);
    const uint8_t* blk = page < 0 ? nullptr : c.block(page, side, head, D);
    if (side == 0) {
      // 16 bytes of a row a lane, so that 64 consecutive values leave together
      constexpr int N = 16 / sizeof(T), PER = 64 / N;
#pragma unroll
      for (int i = 0; i < 16 * D / (64 * N); ++i) {
        const int u = i * 64 + lane, ch = u / (16 * PER), t = u / PER % 16, at = u % PER * N, s = low + t;
        uint32_t w[N / 4] = {};
        if (blk) __builtin_memcpy(w, blk + u * N, N);
        float x[N];
#pragma unroll
        for (int j = 0; j < N / 4; ++j) kv8_numbers<FMT>(w[j], x + 4 * j);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= scale;
        if (s < start || s >= end) continue;
        T* p = base + (rows.first + (s - start)) * stride + ch * 64 + at;
        rows_out(p, x);
      }
    } else {
      // a quad's four tokens of 16 bytes of a row a lane
      constexpr int N = 16 / sizeof(T), PER = 64 / N;
#pragma unroll
      for (int i = 0; i < (4 * D / N + 63) / 64; ++i) {
        const int u = i * 64 + lane, ch = u / (4 * PER), quad = u / PER % 4, at = u % PER * N;
        if (u >= 4 * D / N) break;
        u32x4 w[N / 4] = {};
        if (blk)
#pragma unroll
          for (int j = 0; j < N / 4; ++j) w[j] = reinterpret_cast<const u32x4*>(blk + u * N * 4)[j];
        float x[4 * N];
#pragma unroll
        for (int j = 0; j < N; ++j) kv8_numbers<FMT>(w[j / 4][j & 3], x + 4 * j);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int s = low + 4 * quad + t;
          if (s < start || s >= end) continue;
          float y[N];
#pragma unroll
          for (int j = 0; j < N; ++j) y[j] = x[4 * j + t] * scale;
          T* p = base + (rows.first + (s - start)) * stride + ch * 64 + at;
          rows_out(p, y);
        }
      }
    }
  }
}

// ---- eviction ----
// fp32 as an integer of the same order; NaN below everything
__device__ __forceinline__ uint32_t order_of(float m) {
  const uint32_t b = __builtin_bit_cast(uint32_t, m);
  if (m != m) return 0u;
  if (m == 0.f) return 0x80000000u;                                   // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// the sum of the lanes up to this one
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);      // from 1, 2, 4 and 8 lanes before, within sixteen
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);     // lane 15 to the second sixteen, 47 to the fourth
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);     // lane 31 to the upper half
  return v;
}
// flags of the lanes before this one, on top of n
__device__ __forceinline__ int lanes_before(uint64_t mask, int n) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, n)); }

// Which tokens stay: one workgroup an (entry, head).  Three histograms over 11, 11 and 10 bits of the weights' order give the lightest weight that stays among those
// between the first and the last tokens; then every wave counts, and after a barrier writes, the slots that stay of a run of its own, in order: of equal weights the
// lowest slots.  11 bits reach into the mantissa: weights share few exponents, and counts of one address are taken in turn.  Bound by what few workgroups issue, so the
// weights are fetched once, through their pages, 16 bytes a lane, and kept in shared memory where they fit (36 864 tokens; of those beyond, every pass fetches
// them again), and no pass asks where the first and last tokens are.  8 entries of up to 32 000 tokens and 8 heads: 24 us, 8 of them until the weights are there and
// counted; 2000 tokens 8.6 us, 1 of them a histogram's barriers.
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64, kPickCached = 36864;
constexpr uint32_t kAlways = 0xFFFFFFFFu;   // in the place of a weight's order, which never has it: the first and last tokens, and what lies behind the last
__global__ __launch_bounds__(kPickThreads) void kv8_pick_kernel(Kv8 c, const float* mass, int64_t mass_stride, const int32_t* lens, int budget, int keep_first,
                                                                int keep_last, int cached, int32_t* kept) {
  extern __shared__ u32x4 s_order[];
  __shared__ uint32_t hist[2048];
  __shared__ __attribute__((aligned(16))) int s_sure[kPickWaves], s_ties[kPickWaves], s_sum[kPickWaves];
  __shared__ uint32_t s_bits;
  __shared__ int s_left;
  const int e = blockIdx.y, head = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = c.tokens(e, lens[e]);
  int32_t* out = kept + ((int64_t)e * c.kv_heads + head) * budget;
  if (len <= budget) {
    for (int i = tid; i < budget; i += kPickThreads) out[i] = i < len ? i : -1;
    return;
  }
  // the weights of N fours of slots (from multiples of 4: of one page), page ids and weights each in one go: what is not there is read from the table's and the
  // cache's first place and left out
  const int first = c.indptr[e], pages = c.indptr[e + 1] - first;
  const int lo = keep_first, hi = len - keep_last, chosen = budget - keep_first - keep_last;
  constexpr int N = 4;
  auto fetch = [&](auto slot, u32x4 (&w)[N]) {
    int page[N];
    f32x4 m[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int block = slot(i) / kKv8Page, at = first + block;
      const bool there = block < pages && (unsigned)at < (unsigned)c.n_ids;
      const int id = c.ids[there ? at : 0];
      page[i] = there && (unsigned)id < (unsigned)c.n_pages ? id : -1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) __builtin_memcpy(&m[i], mass + max(page[i], 0) * mass_stride + head * kKv8Page + slot(i) % kKv8Page, 16);   // on 4 bytes
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = slot(i) + j;
        w[i][j] = s < lo || s >= hi ? kAlways : page[i] < 0 ? 0u : order_of(m[i][j]);
      }
  };
  auto of_waves_before = [&](const int (&x)[kPickWaves]) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) sum += i < wave ? x[i] : 0;
    return sum;
  };
  const int held = min(len, cached);       // slots whose weights are in shared memory (a multiple of 4, or all); the others' are fetched again
  for (int i = tid; i < 2048; i += kPickThreads) hist[i] = 0;
  __syncthreads();
  constexpr int kStep = 4 * kPickThreads;
  for (int s0 = 4 * tid; s0 < len; s0 += N * kStep) {
    u32x4 w[N];
    fetch([&](int i) { return s0 + i * kStep; }, w);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = s0 + i * kStep;
      if (s < held) s_order[s / 4] = w[i];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w[i][j] != kAlways) atomicAdd(&hist[w[i][j] >> 21], 1u);
    }
  }
  uint32_t bits = chosen > 0 ? 0u : kAlways - 1;   // of the lightest weight that stays: its upper bits so far
  int left = chosen;                       // tokens still to be found that have those
  if (chosen > 0) {
    for (int done = 0; done < 32; done += 11) {
      const int width = min(11, 32 - done), shift = 32 - done - width;
      if (done > 0) {
        for (int i = tid; i < 2048; i += kPickThreads) hist[i] = 0;
        __syncthreads();
      }
      const uint32_t mask = done == 0 ? 0u : 0xFFFFFFFFu << (32 - done);
      if (done > 0) {                      // the first is counted as the weights arrive
        auto count = [&](const u32x4& w) {
          bool here[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) here[j] = (w[j] & mask) == bits;     // never one that always stays
          if (here[0] | here[1] | here[2] | here[3])
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (here[j]) atomicAdd(&hist[(w[j] >> shift) & 2047 >> (11 - width)], 1u);
        };
#pragma unroll 4
        for (int s = 4 * tid; s < held; s += kStep) count(s_order[s / 4]);
        for (int s0 = held + 4 * tid; held < len && s0 < len; s0 += N * kStep) {
          u32x4 w[N];
          fetch([&](int i) { return s0 + i * kStep; }, w);
#pragma unroll
          for (int i = 0; i < N; ++i) count(w[i]);
        }
      }
      __syncthreads();
      // thread t: digits 2047 - 2 t and 2046 - 2 t; how many weights have a larger digit
      const int a = (int)hist[2047 - 2 * tid], b = (int)hist[2046 - 2 * tid];
      int sum = wave_scan(a + b);
      if (lane == 63) s_sum[wave] = sum;
      __syncthreads();
      sum += of_waves_before(s_sum);
      const int above = sum - a - b;
      if (above < left && left <= sum) {   // one thread: the counts reach `left` in its two digits
        const bool second = left > above + a;
        s_bits = bits | (uint32_t)(2047 - 2 * tid - second) << shift;
        s_left = left - above - (second ? a : 0);
      }
      __syncthreads();
      bits = s_bits;
      left = s_left;
    }
  }
  __syncthreads();
  // A wave's run is whole steps of its walk.  What the last one sees behind the last token always stays, or is the last token again: it comes when all places are taken.
  constexpr int U = 2;                     // fours of slots a lane at a time: two of shared memory, or N through the pages
  const int unit = 256 * (held < len ? N : U), run = (len + kPickWaves * unit - 1) / (kPickWaves * unit) * unit, from = min(wave * run, len), to = min(from + run, len);
  const int near = held == len ? to : min(to, from + max(held - from, 0) / unit * unit);      // of the run, in shared memory
  auto look = [&](int s, const u32x4& w, auto&& each) {
    uint64_t sure[4], tie[4];              // of the wave's lanes, of each of their slots
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sure[j] = __builtin_amdgcn_ballot_w64(w[j] > bits);
      tie[j] = __builtin_amdgcn_ballot_w64(w[j] == bits);
    }
    each(s, sure, tie);
  };
  auto walk = [&](auto&& each) {
    int at = from;
    for (; at < near; at += 256 * U) {
      u32x4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = s_order[min(at + u * 256 + 4 * lane, held - 1) / 4];
#pragma unroll
      for (int u = 0; u < U; ++u) look(at + u * 256 + 4 * lane, w[u], each);
    }
    for (; at < to; at += 256 * N) {
      u32x4 w[N];
      fetch([&](int i) { return at + i * 256 + 4 * lane; }, w);
#pragma unroll
      for (int i = 0; i < N; ++i) look(at + i * 256 + 4 * lane, w[i], each);
    }
  };
  int sures = 0, ties = 0;
  walk([&](int, const uint64_t (&sure)[4], const uint64_t (&tie)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sures += __popcll(sure[j]);
      ties += __popcll(tie[j]);
    }
  });
  if (lane == 0) { s_sure[wave] = sures; s_ties[wave] = ties; }
  __syncthreads();
  int tied = of_waves_before(s_ties), at = of_waves_before(s_sure) + min(tied, left);      // ties met, and tokens that stay, in the slots before
  walk([&](int s, const uint64_t (&sure)[4], const uint64_t (&tie)[4]) {
    uint64_t stays[4];
    int before = tied;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      stays[j] = sure[j];
      before = lanes_before(tie[j], before);
    }
    if (tie[0] | tie[1] | tie[2] | tie[3]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool here = tie[j] >> lane & 1;
        stays[j] |= __builtin_amdgcn_ballot_w64(here && before < left);
        before += here;
        tied += __popcll(tie[j]);
      }
    }
    int put = at;
#pragma unroll
    for (int j = 0; j < 4; ++j) put = lanes_before(stays[j], put);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool here = stays[j] >> lane & 1;
      if (here && put < budget) out[put] = s + j;
      put += here;
      at += __popcll(stays[j]);
    }
  });
}

// The kept tokens into fresh pages: a wave a block's keys, another its values.  A block's exponent is the largest of its tokens', whose codes stay as they are.
// Bound by bytes: tokens that stay are a quarter here and there, and a value block's 16 bytes hold four tokens (8 entries of up to 32 000 -> 8000 of 8 x 128: 78 us).
template <int FMT, int D>
__global__ __launch_bounds__(128) void kv8_move_kernel(Kv8 c, const int32_t* dst_indptr, const int32_t* dst_ids, int n_dst_ids, float* mass, int64_t mass_stride,
                                                       const int32_t* lens, int budget, const int32_t* kept) {
  const int e = blockIdx.z, head = blockIdx.y, side = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const int len = min(c.tokens(e, lens[e]), budget);
  const int32_t* from = kept + ((int64_t)e * c.kv_heads + head) * budget;
  Kv8 to = c;
  to.indptr = dst_indptr;
  to.ids = dst_ids;
  to.n_ids = n_dst_ids;
  for (int b = blockIdx.x; b < (len + kKv8Page - 1) / kKv8Page; b += gridDim.x) {
    const int dst = to.page(e, b);
    if (dst < 0) continue;
    // lane n of every sixteen: where token n comes from
    const int i = b * kKv8Page + n, slot = i < len ? from[i] : -1, src = slot < 0 ? -1 : c.page(e, slot / kKv8Page), t = slot & 15;
    const int was = src < 0 ? kKv8LeastExp : exp_of(*c.scale(src, side, head));
    int ex = was;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) ex = max(ex, __shfl_xor(ex, d, 64));
    if (side == 0 && q == 0) mass[dst * mass_stride + head * kKv8Page + n] = src < 0 ? 0.f : mass[src * mass_stride + head * kKv8Page + t];
    uint8_t* blk = to.block(dst, side, head, D);
    if (lane == 0) *to.scale(dst, side, head) = pow2f(ex);
    int src4[4], t4[4], was4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      src4[j] = __shfl(src, 4 * q + j, 64);
      t4[j] = __shfl(t, 4 * q + j, 64);
      was4[j] = __shfl(was, 4 * q + j, 64);
    }
    // every load at once; a token that is not there: the first page's bytes, left out
    if (side == 0) {
      u32x4 w[D / 64];
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) w[ch] = *reinterpret_cast<const u32x4*>(c.block(max(src, 0), 0, head, D) + unit_at(0, ch, t, q));
      const float by = pow2f(was - ex);
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        if (src < 0) w[ch] = u32x4{0, 0, 0, 0};
        if (was != ex) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float y[4];
            kv8_numbers<FMT>(w[ch][k], y);
#pragma unroll
            for (int m = 0; m < 4; ++m) y[m] *= by;
            w[ch][k] = kv8_codes<FMT>(y);
          }
        }
        *reinterpret_cast<u32x4*>(blk + unit_at(0, ch, n, q)) = w[ch];
      }
    } else {
      u32x4 g[D / 64][4];
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch)
#pragma unroll
        for (int j = 0; j < 4; ++j) g[ch][j] = *reinterpret_cast<const u32x4*>(c.block(max(src4[j], 0), 1, head, D) + unit_at(1, ch, n, t4[j] >> 2));
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        u32x4 w = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t one = 0;                // this token's byte of each of the four values
#pragma unroll
          for (int k = 0; k < 4; ++k) one |= (g[ch][j][k] >> (8 * (t4[j] & 3)) & 255u) << (8 * k);
          if (src4[j] < 0) one = 0;
          if (was4[j] != ex) {
            float y[4];
            kv8_numbers<FMT>(one, y);
#pragma unroll
            for (int m = 0; m < 4; ++m) y[m] *= pow2f(was4[j] - ex);
            one = kv8_codes<FMT>(y);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] |= (one >> (8 * k) & 255u) << (8 * j);
        }
        *reinterpret_cast<u32x4*>(blk + unit_at(1, ch, n, q)) = w;
      }
    }
  }
}

static pegainfer_status_t append_rows(const pegainfer_kv8_cache* cache, float* mass, int64_t mass_page_stride, const void* k, const void* v, int64_t k_row_stride,
                                      int64_t v_row_stride, const int32_t* row0, const int32_t* starts, int32_t n_rows, int32_t max_rows, int32_t dtype,
                                      pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || n_rows < 0 || max_rows < 0 || (dtype != kDtBf16 && dtype != kDtF32)) return PK_BAD;
  if (n_rows == 0 || cache->n_entries == 0) return 0;
  const int64_t width = (int64_t)cache->kv_heads * cache->dim, unit = dtype == kDtBf16 ? 8 : 4;
  if (!k || !v || !row0 || !starts || !host_aligned16(k) || !host_aligned16(v) || k_row_stride < width || v_row_stride < width || k_row_stride % unit || v_row_stride % unit)
    return PK_BAD;
  const Kv8 c = kv8_of(cache);
  const dim3 grid(std::min(max_rows, n_rows) / kKv8Page + 2, c.kv_heads, c.entries);
  kv8_by(dtype, cache->format, cache->dim, [&](auto* t, auto fmt, auto dim) {
    using T = std::remove_pointer_t<decltype(t)>;
    kv8_append_kernel<T, fmt(), dim()><<<grid, 128, 0, as_stream(stream)>>>(c, mass, mass_page_stride, static_cast<const T*>(k), static_cast<const T*>(v), k_row_stride,
                                                                            v_row_stride, row0, starts, n_rows);
  });
  return (pegainfer_status_t)hipGetLastError();
}

}  // namespace pk

using namespace pk;

extern "C" {

pegainfer_status_t pegainfer_kv8_append(const pegainfer_kv8_cache* cache, const void* k, const void* v, int64_t k_row_stride, int64_t v_row_stride,
                                        const int32_t* row0, const int32_t* starts, int32_t n_rows, int32_t max_rows, int32_t dtype, pegainfer_stream_t stream) {
  return append_rows(cache, nullptr, 0, k, v, k_row_stride, v_row_stride, row0, starts, n_rows, max_rows, dtype, stream);
}

pegainfer_status_t pegainfer_kv8_append_weighed(const pegainfer_kv8_cache* cache, float* mass, int64_t mass_page_stride, const void* k, const void* v, int64_t k_row_stride,
                                                int64_t v_row_stride, const int32_t* row0, const int32_t* starts, int32_t n_rows, int32_t max_rows, int32_t dtype,
                                                pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || !mass || mass_page_stride < (int64_t)cache->kv_heads * kKv8Page) return PK_BAD;
  return append_rows(cache, mass, mass_page_stride, k, v, k_row_stride, v_row_stride, row0, starts, n_rows, max_rows, dtype, stream);
}

pegainfer_status_t pegainfer_kv8_read(const pegainfer_kv8_cache* cache, const int32_t* row0, const int32_t* starts, void* k, void* v, int32_t n_rows, int32_t max_rows,
                                      int32_t dtype, pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || n_rows < 0 || max_rows < 0 || (dtype != kDtBf16 && dtype != kDtF32)) return PK_BAD;
  if (n_rows == 0 || cache->n_entries == 0) return 0;
  if (!row0 || !starts || !k || !v || !host_aligned16(k) || !host_aligned16(v)) return PK_BAD;
  const Kv8 c = kv8_of(cache);
  const dim3 grid(std::min(max_rows, n_rows) / kKv8Page + 2, c.kv_heads, c.entries);
  kv8_by(dtype, cache->format, cache->dim, [&](auto* t, auto fmt, auto dim) {
    using T = std::remove_pointer_t<decltype(t)>;
    kv8_read_kernel<T, fmt(), dim()><<<grid, 128, 0, as_stream(stream)>>>(c, static_cast<T*>(k), static_cast<T*>(v), row0, starts, n_rows);
  });
  return (pegainfer_status_t)hipGetLastError();
}

pegainfer_status_t pegainfer_kv8_evict(const pegainfer_kv8_cache* cache, float* mass, int64_t mass_page_stride, const int32_t* lens, const int32_t* dst_indptr,
                                       const int32_t* dst_ids, int32_t n_dst_ids, int32_t budget, int32_t keep_first, int32_t keep_last, int32_t max_len, int32_t* kept,
                                       pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || budget < 1 || keep_first < 0 || keep_last < 0 || keep_first > budget - keep_last || n_dst_ids < 0 || max_len < 0) return PK_BAD;
  if (cache->n_entries == 0) return 0;
  if (!mass || !lens || !dst_indptr || (!dst_ids && n_dst_ids > 0) || !kept || mass_page_stride < (int64_t)cache->kv_heads * kKv8Page) return PK_BAD;
  const Kv8 c = kv8_of(cache);
  const int cached = (std::min(max_len, kPickCached) + 3) / 4 * 4;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kv8_pick_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kPickCached * 4) != hipSuccess) return PK_BAD;
  kv8_pick_kernel<<<dim3(c.kv_heads, c.entries), kPickThreads, cached * 4, as_stream(stream)>>>(c, mass, mass_page_stride, lens, budget, keep_first, keep_last, cached, kept);
  const dim3 grid(std::max(1, ceil_div(std::min(budget, max_len), kKv8Page)), c.kv_heads, c.entries);
  kv8_by(kDtBf16, cache->format, cache->dim, [&](auto*, auto fmt, auto dim) {
    kv8_move_kernel<fmt(), dim()><<<grid, 128, 0, as_stream(stream)>>>(c, dst_indptr, dst_ids, n_dst_ids, mass, mass_page_stride, lens, budget, kept);
  });
  return (pegainfer_status_t)hipGetLastError();
}

}  // extern "C"
