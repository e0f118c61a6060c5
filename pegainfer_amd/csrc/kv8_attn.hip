// Softmax attention over the 8-bit paged cache, and the weight that every cached token gets.
//
//   o[r, h] = sum_j p_j v_j,  p = softmax_j(scale q[r, h] . k_j) over the slots j <= starts[e] + i of row i of entry e
//   mass_out[j, g] = keep mass[j, g] + sum over the entry's rows r and the query heads h of kv head g of p_j[r, h]
#include <algorithm>

#include "kv8_host.h"

namespace pk {

__device__ __forceinline__ f32x4 mfma16(const bf16x8_t& a, const bf16x8_t& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN among them does not count
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Results of matrix instructions that an assembly statement is the first to read: the compiler puts the wait states of that read in front of instructions that it
// knows, not of assembly (16x16x32: 12 at most), so they stand here, tied to the registers.
template <int NT, int KB>
__device__ __forceinline__ void settle(f32x4 (&s)[NT][KB]) {
  static_assert((NT * KB) % 2 == 0 && (NT * KB <= 2 || (NT * KB) % 8 == 0), "two or eight registers a statement");
  f32x4* p = &s[0][0];
  if constexpr (NT * KB == 2) asm("s_nop 15" : "+v"(p[0]), "+v"(p[1]));
  else
#pragma unroll
    for (int i = 0; i < NT * KB; i += 8)
      asm("s_nop 15" : "+v"(p[i]), "+v"(p[i + 1]), "+v"(p[i + 2]), "+v"(p[i + 3]), "+v"(p[i + 4]), "+v"(p[i + 5]), "+v"(p[i + 6]), "+v"(p[i + 7]));
}
// the other half's (of 32) and the other row's (of 16) value, without a trip through shared memory; s_nop: the wait states between a VALU write and the swap.  In
// assembly because the swap wants two registers, and the builtin given one value twice may be folded to one.
template <typename Op>
__device__ __forceinline__ float across_quad(float v, Op op) {
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  a = op(a, b);
  b = a;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return op(a, b);
}
// over the four lanes that hold a row's scores
__device__ __forceinline__ float quad_max(float v) { return across_quad(v, [](float x, float y) { return fmaxf(x, y); }); }
__device__ __forceinline__ float quad_sum(float v) { return across_quad(v, [](float x, float y) { return x + y; }); }
// The maximum that a row's weights are taken against moves only when a score passes it by a factor of 2^kSlack, so that most steps need no exchange between lanes
// and no rescaling.  Not by more: the maximum's own key has a weight of 1 (in prompts' unmasked steps but for the rounding of its score, 2^-24 of it, which bf16 takes
// off again for scores below 2^15) and a key above it at most 2, so no key whose weight is rounded to bf16 has over two thirds of a row, and one with almost all of it
// gives its values.  16 rows x 500 keys to 256 rows x 20000: outputs off by 1.64 to 1.73e-3 of their norm, 1.62
// to 1.71e-3 with none, 1.72 to 1.97e-3 with 8; 2048 rows over 8192 tokens 255 us, 258 with none, 251 with 8.
constexpr float kSlack = 1.f;

struct AttnArgs {
  Kv8 c;
  const void* q;
  int64_t q_stride, out_stride;
  const int32_t *row0, *starts;
  int n_rows, group, heads, n_split, split_blocks;
  float scale_log2;
  void* out;
  float* lse;            // [n_rows][heads], log2 of the sum of exp(scores); NULL: not wanted
  float *part_o, *part_ml;   // n_split > 1: [n_rows][heads][n_split][D] and [2] (running maximum, sum)
  float* scores;         // [n_ids][kv_heads][score_rows][16] of entries of up to score_rows <= 16 query rows a kv head, for the weights; NULL: not wanted
  int score_rows;
  int round, snake;      // pieces of work of an entry and head that one workgroup a compute unit takes; whether the second round goes from the short to the long
};

// the queries' rows of a kv head, (token, head of the group) in order; a row behind the last is the last again
struct QueryRow { int row, head, far; bool real; };   // far: the last slot that it sees
__device__ __forceinline__ QueryRow query_row(int rr, int total, int group, const RowSpan& rows, int start, int kv_head) {
  const int r = min(rr, total - 1), tok = r / group;
  return {rows.first + tok, kv_head * group + r - tok * group, start + tok, rr < total};
}

constexpr int kPromptRows = 128;

// a lane's part of a row's result: the output, or what a split leaves of it
template <typename T, int D>
__device__ __forceinline__ void put_row(const AttnArgs& a, const QueryRow& r, int split, int g, float m, float l, const f32x4 (&o)[D / 16]) {
  const bool some = l > 0.f || l != l;
  const float inv = a.n_split > 1 ? 1.f : some ? 1.f / l : 0.f;   // no key: zeros
  const int64_t rh = (int64_t)r.row * a.heads + r.head;
  auto put = [&](auto* op) {
    using O = std::remove_pointer_t<decltype(op)>;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = o[4 * c + j][i] * inv;
      Vec8<O>::store(op + g * 16 + c * 64, x);
      Vec8<O>::store(op + g * 16 + c * 64 + 8, x + 8);
    }
  };
  if (a.n_split > 1) {
    if (some) put(a.part_o + (rh * a.n_split + split) * D);
    if (g == 0) *reinterpret_cast<f32x2*>(a.part_ml + (rh * a.n_split + split) * 2) = f32x2{m, l};
  } else {
    put(static_cast<T*>(a.out) + r.row * a.out_stride + (int64_t)r.head * D);
    if (a.lse && g == 0) a.lse[rh] = some ? m + __log2f(l) : INFINITY;
  }
}

struct MassArgs {
  const float* mass;
  float *out, *part;     // part [n_slice][n_ids][kv_heads][16]
  int64_t mass_stride, out_stride;
  float keep;
  int n_slice;
};
__device__ __forceinline__ void put_mass(const MassArgs& w, int page, int at, float x) {
  // 0 means without what was there, whatever that is
  w.out[page * w.out_stride + at] = w.keep == 0.f ? x : fmaf(w.keep, w.mass[page * w.mass_stride + at], x);
}

// log2 of a row's sum of exp(scores) from its splits' states, a wave's lanes a split each
__device__ __forceinline__ float lse_of_splits(const AttnArgs& a, int64_t rh, int lane) {
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + rh * a.n_split;
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < a.n_split; i += 64) m = fmaxf(m, ml[i].x);
  m = wave_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  for (int i = lane; i < a.n_split; i += 64) l += ml[i].y * exp2_of(ml[i].x - base);     // of a split without a key: 0 times exp2(-infinity)
  l = wave_sum(l);
  return l > 0.f || l != l ? m + __log2f(l) : INFINITY;
}

// The same of lane (n, g)'s row n, by the four lanes that have it
__device__ __forceinline__ float lse_of_row(const AttnArgs& a, int64_t rh, int g) {
  if (a.n_split == 1) return a.lse[rh];
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + rh * a.n_split;
  float m = -INFINITY, l = 0.f;
  for (int i = g; i < a.n_split; i += 4) m = fmaxf(m, ml[i].x);
  m = quad_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  for (int i = g; i < a.n_split; i += 4) l += ml[i].y * exp2_of(ml[i].x - base);
  l = quad_sum(l);
  return l > 0.f || l != l ? m + __log2f(l) : INFINITY;
}

// What the tokens of an entry weigh that has more rows than the call said, and so no scores, by workgroup z of `ways`: every wave two blocks (fp32: one; more
// take registers that a step's waves want), sixteen rows at a time, their products taken again.  A portion of 256
// rows of 128 values among 31 single ones that the hint is made for, 8 heads: 184 us over 300 tokens, 105 of them the attention, and 656, 521 of them, over 4000
// (a thread a token took 3447 and 5169; with the portion's rows as the hint 52 and 257).
template <typename T, int FMT, int D>
__device__ __forceinline__ void rows_mass(const AttnArgs& a, const MassArgs& w, int e, int head, const RowSpan& rows, int start, int z, int ways) {
  constexpr int NP = kv8_parts<T>(), C = D / 64, B = sizeof(T) == 2 ? 2 : 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int len = a.c.tokens(e, start + rows.n), total = rows.n * a.group;
  for (int b0 = (z * 4 + wave) * B; b0 * kKv8Page < len; b0 += ways * 4 * B) {
    f32x4 sum[B];
#pragma unroll
    for (int h = 0; h < B; ++h) sum[h] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int first = (int)((int64_t)max(b0 * kKv8Page - start, 0) * a.group / 16);       // the first sixteen with a row that sees one of the blocks
    for (int tile = first; tile * 16 < total; ++tile) {
      const QueryRow r = query_row(tile * 16 + n, total, a.group, rows, start, head);
      const float lse = lse_of_row(a, (int64_t)r.row * a.heads + r.head, g), off = r.real ? lse : INFINITY;     // a row behind the last weighs nothing
      const T* qp = static_cast<const T*>(a.q) + r.row * a.q_stride + (int64_t)r.head * D + g * 16;
      f32x4 s[B];
#pragma unroll
      for (int h = 0; h < B; ++h) s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < C; ++c) {
        bf16x8_t q[2][NP];
        kv8_query(qp + c * 64, q[0]);
        kv8_query(qp + c * 64 + 8, q[1]);
#pragma unroll
        for (int h = 0; h < B; ++h) {
          const u32x4 k = *reinterpret_cast<const u32x4*>(a.c.block(max(a.c.page(e, b0 + h), 0), 0, head, D) + c * 1024 + n * 64 + g * 16);
          const bf16x8_t k0 = kv8_operand<FMT>(k.x, k.y), k1 = kv8_operand<FMT>(k.z, k.w);
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) {
            s[h] = mfma16(k0, q[0][p], s[h]);
            s[h] = mfma16(k1, q[1][p], s[h]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < B; ++h) {
        const float ks = *a.c.scale(max(a.c.page(e, b0 + h), 0), 0, head) * a.scale_log2;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[h][i] += (b0 + h) * kKv8Page + 4 * g + i <= r.far ? exp2_of(fmaf(s[h][i], ks, -off)) : 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < B; ++h) {
      const int page = a.c.page(e, b0 + h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = row16_sum(sum[h][i]);
        const int t = 4 * g + i;
        if (n == i && page >= 0 && (b0 + h) * kKv8Page + t < len) put_mass(w, page, head * kKv8Page + t, x);
      }
    }
  }
}

// What an entry's tokens weigh in a step, a thread a token, by workgroup z of `ways`, from the scores that the attention left (4 bytes a row beside D of the keys) and the
// rows' log-sums.  Of up to 16 rows whatever the head, against keys and rows multiplied again (kv8_mass_kernel), 16 rows of each: 16 entries x 4096 tokens of 64 values 40 us
// and 57, of 128 53 and 69, of 256 43 and 62; x 1000 tokens 19, 23, 32 and 20, 24, 29; a single row 25, 35, 31 and 56, 68, 60.
constexpr int kStepRows = 16;
template <typename T, int FMT, int D>
__device__ __forceinline__ void step_mass(const AttnArgs& a, const MassArgs& w, int e, int head, const RowSpan& rows, int start, int z, int ways, float (&s_lse)[kStepRows]) {
  const int len = a.c.tokens(e, start + rows.n), first_block = a.c.indptr[e], total = rows.n * a.group, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (total > a.score_rows) return rows_mass<T, FMT, D>(a, w, e, head, rows, start, z, ways);
  if (z * 256 >= len) return;
  auto row_head = [&](int rr) { const QueryRow r = query_row(rr, total, a.group, rows, start, head); return (int64_t)r.row * a.heads + r.head; };
  for (int rr = wave; rr < total; rr += 4) {
    const float x = a.n_split > 1 ? lse_of_splits(a, row_head(rr), lane) : a.lse[row_head(rr)];
    if (lane == 0) s_lse[rr] = x;
  }
  __syncthreads();
  for (int slot0 = z * 256; slot0 < len; slot0 += ways * 256) {
    const int slot = slot0 + threadIdx.x, block = slot / kKv8Page, t = slot % kKv8Page, page = slot < len ? a.c.page(e, block) : -1;
    if (page < 0) continue;
    const float* s = a.scores + (((int64_t)first_block + block) * a.c.kv_heads + head) * a.score_rows * kKv8Page + t;
    float x = 0.f;
#pragma unroll 4
    for (int rr = 0; rr < total; ++rr) x += exp2_of(s[rr * kKv8Page] - s_lse[rr]);
    put_mass(w, page, head * kKv8Page + t, x);
  }
}

// Blocks a wave takes at a time, and waves of a SIMD: what the registers hold without spilling.  Four blocks of 128 values and two row tiles spill, and are slower by
// a tenth than two blocks (8 entries of 16 rows over 4000 tokens: 28.2 and 26.4 us); with one tile four are faster over short contexts (1024 tokens: 9.8 and 10.3 us)
// and two over longer ones of few entries (8 x 4096: 16.2 and 15.2).
template <typename T, int D, int NT> constexpr int attn_kb() { return D == 64 ? (sizeof(T) == 2 || NT == 1 ? 4 : 2) : D == 128 && sizeof(T) == 2 && NT == 1 ? 4 : 2; }
template <typename T, int D, int NT> constexpr int attn_waves() {
  return D == 256 ? (sizeof(T) == 2 && NT == 1 ? 2 : 1) : sizeof(T) == 4 && D * NT == 256 ? 1 : D * NT == 64 && sizeof(T) == 2 ? 3 : 2;
}

// One workgroup of four waves: NT tiles of sixteen query rows of a kv head over a run of key blocks.  The blocks are dealt to the waves KB at a time, whose states
// meet in shared memory at the end, so that no key is loaded or widened twice in a workgroup.  Scores are computed transposed (keys x rows): a lane then holds four
// keys' scores of one row, exactly what the second product wants from it.  The next keys are on their way while the weights are made, the next values while
// the next scores are.
// ONCE: the rows are one tile, so nobody reads the keys again and they pass the caches by (32 x 8192 tokens int8: 78 -> 70 us, 4.8 TB/s).
// FEW: a step over so few tokens that the workgroup, which has seen them all, gives them their weights as well, without a second launch (100 tokens: captured 9.5 -> 8.4 us,
// called one by one 14.2 -> 12.0; over 1024 tokens the four walks through the scores take 1.5 us more than the launch).  An instance of its own: at its end the others lose 0.6 us.
template <typename T, int FMT, int D, int NT, bool ONCE, bool FEW>
__global__ __launch_bounds__(256, (attn_waves<T, D, NT>())) void kv8_attn_kernel(AttnArgs a, MassArgs w) {
  constexpr int NP = kv8_parts<T>(), C = D / 64, KB = attn_kb<T, D, NT>(), W = 4;
  constexpr bool kScaled = FMT == kE4m3;   // the conversion takes the block's scale along; int8 scales scores and weights instead
  __shared__ f32x4 s_o[W / 2][D / 16][64];
  __shared__ float s_m[W / 2][16], s_l[W / 2][16], s_lse[FEW ? kStepRows : 1];
  const int e = (blockIdx.y + blockIdx.z / a.n_split / a.round) % gridDim.y, head = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  const int len = start + rows.n, n_tiles = (total + 16 * NT - 1) / (16 * NT), split = blockIdx.z % a.n_split, step = gridDim.z / a.n_split;
  for (int at = blockIdx.z / a.n_split; at < n_tiles; at += step) {
    const int tile = a.snake && at >= a.round ? at - a.round : n_tiles - 1 - at;     // the rows that see most first
    QueryRow r[NT];
    bf16x8_t qf[NT][C][2][NP];
    float m[NT], l[NT];
    f32x4 o[NT][D / 16];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      r[t] = query_row((tile * NT + t) * 16 + n, total, a.group, rows, start, head);
      const T* qp = static_cast<const T*>(a.q) + r[t].row * a.q_stride + (int64_t)r[t].head * D + g * 16;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        kv8_query(qp + c * 64, qf[t][c][0]);
        kv8_query(qp + c * 64 + 8, qf[t][c][1]);
      }
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // slots that every row of the tiles sees, and that any does
    const int all_see = tile * NT * 16 / a.group + start, any_sees = min((tile + 1) * NT * 16 - 1, total - 1) / a.group + start;
    const int blocks = min(any_sees / kKv8Page + 1, a.c.blocks(e)), per = max(a.split_blocks, (blocks + a.n_split - 1) / a.n_split);
    const int b_lo = split * per, b_hi = min(blocks, b_lo + per);
    // lane i: block i of a run of 64; the pages of a run are looked up two runs ahead, their scales one
    auto page_of = [&](int run) { return run + lane < b_hi ? a.c.page(e, run + lane) : -1; };
    auto scale_of = [&](int page, int side) { return page < 0 ? 0.f : *a.c.scale(page, side, head); };
    int pid = page_of(b_lo), next = page_of(b_lo + 64);
    float ks = scale_of(pid, 0), vs = scale_of(pid, 1);
    u32x4 kw[KB][C], vw[KB][C];
    auto load = [&](int side, int pages, int i, u32x4 (&w)[KB][C]) {
#pragma unroll
      for (int h = 0; h < KB; ++h) {
        const int page = max(__builtin_amdgcn_readlane(pages, i * KB + h), 0);     // one that is not there: page 0's bytes, masked below
        const uint8_t* p = a.c.block(page, side, head, D) + (side == 0 ? n * 64 + g * 16 : g * 256 + n * 16);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const u32x4* from = reinterpret_cast<const u32x4*>(p + c * 1024);
          w[h][c] = ONCE ? __builtin_nontemporal_load(from) : *from;
        }
      }
    };
    auto lane_of = [](float v, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
    if (wave * KB < b_hi - b_lo) {
      load(0, pid, wave, kw);
      load(1, pid, wave, vw);
    }
    for (int run = b_lo; run < b_hi; run += 64) {
      const float next_ks = scale_of(next, 0), next_vs = scale_of(next, 1);
      const int after = page_of(run + 128);
      const uint64_t there = __builtin_amdgcn_ballot_w64(pid >= 0);
      const int groups = (min(b_hi - run, 64) + KB - 1) / KB;
      const bool more = run + 64 + wave * KB < b_hi;     // the wave has a group in the next run
      for (int i = wave; i < groups; i += W) {
        const int slot0 = (run + i * KB) * kKv8Page;
        f32x4 s[NT][KB];
#pragma unroll
        for (int h = 0; h < KB; ++h) {
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
          const float kscale = lane_of(ks, i * KB + h);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const bf16x8_t k0 = kv8_operand<FMT>(kw[h][c].x, kw[h][c].y, kscale), k1 = kv8_operand<FMT>(kw[h][c].z, kw[h][c].w, kscale);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                s[t][h] = mfma16(k0, qf[t][c][0][p], s[t][h]);
                s[t][h] = mfma16(k1, qf[t][c][1][p], s[t][h]);
              }
          }
          const float f = kScaled ? a.scale_log2 : kscale * a.scale_log2;
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][h] *= f;
        }
        if (i + W < groups) load(0, pid, i + W, kw);
        else if (more) load(0, next, wave, kw);
        const uint64_t want = ((1ull << KB) - 1) << (i * KB);
        const bool ragged = slot0 + KB * kKv8Page - 1 > all_see || (there & want) != want;
        if (ragged) {
#pragma unroll
          for (int h = 0; h < KB; ++h) {
            const int end = there >> (i * KB + h) & 1 ? INT32_MAX : -1, at0 = slot0 + h * kKv8Page + 4 * g;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[t][h][j] = at0 + j <= min(r[t].far, end) ? s[t][h][j] : -INFINITY;
            // what lies behind the entry's last token may be any bytes, and 0 times one of them a NaN
            const int here = min(len, end) - at0;
            const uint32_t bytes = here >= 4 ? 0xFFFFFFFFu : here <= 0 ? 0u : 0xFFFFFFFFu >> (32 - 8 * here);
#pragma unroll
            for (int c = 0; c < C; ++c) vw[h][c] &= bytes;
          }
        }
        if constexpr (NT == 1) {
          if (a.scores && total <= a.score_rows && r[0].real) {
            const int64_t first = a.c.indptr[e] + run + i * KB;
#pragma unroll
            for (int h = 0; h < KB; ++h)
              if (there >> (i * KB + h) & 1) *reinterpret_cast<f32x4*>(a.scores + ((((first + h) * a.c.kv_heads + head) * a.score_rows + n) * kKv8Page + 4 * g)) = s[0][h];
          }
        }
        bf16x8_t pf[NT][KB / 2][NP];
        float top[NT], alpha[NT];
        bool moves = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          top[t] = s[t][0][0];
#pragma unroll
          for (int h = 0; h < KB; ++h) top[t] = max3(max3(top[t], s[t][h][0], s[t][h][1]), s[t][h][2], s[t][h][3]);
          moves |= top[t] > m[t] + kSlack;
          alpha[t] = 1.f;
        }
        if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const float mx = quad_max(top[t]), to = mx > m[t] + kSlack ? mx : m[t];
            alpha[t] = to == -INFINITY ? 1.f : exp2_of(m[t] - to);
            m[t] = to;
            l[t] *= alpha[t];
            if constexpr (NP == 1)
#pragma unroll
              for (int d = 0; d < D / 16; ++d) o[t][d] *= alpha[t];
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float base = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
          for (int h = 0; h < KB; h += 2) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              p[j] = exp2_of(s[t][h + j / 4][j & 3] - base);
              l[t] += p[j];
              if (!kScaled) p[j] *= lane_of(vs, i * KB + h + j / 4);
            }
            kv8_split<NP>(p, pf[t][h / 2]);
          }
        }
        // fp32 sums of many keys are added outside the matrix cores, whose accumulation does not round to nearest
        constexpr bool kOutside = NP > 1;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4 x[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = kOutside ? f32x4{0.f, 0.f, 0.f, 0.f} : o[t][4 * c + j];
#pragma unroll
            for (int h = 0; h < KB; h += 2) {
              const bf16x8_t vf = kv8_operand2<FMT>(vw[h][c][j], vw[h + 1][c][j], lane_of(vs, i * KB + h), lane_of(vs, i * KB + h + 1));
#pragma unroll
              for (int k = NP - 1; k >= 0; --k)
#pragma unroll
                for (int t = 0; t < NT; ++t) x[t] = mfma16(vf, pf[t][h / 2][k], x[t]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][4 * c + j] = kOutside ? o[t][4 * c + j] * alpha[t] + x[t] : x[t];
          }
        if (i + W < groups) load(1, pid, i + W, vw);
        else if (more) load(1, next, wave, vw);
      }
      pid = next;
      next = after;
      ks = next_ks;
      vs = next_vs;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] = quad_sum(l[t]);
      // the waves' states into one: the upper half's into the lower's, and so on
#pragma unroll
      for (int half = W / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) s_o[wave - half][i][lane] = o[t][i];
          if (g == 0) { s_m[wave - half][n] = m[t]; s_l[wave - half][n] = l[t]; }
        }
        __syncthreads();
        if (wave < half) {
          const float mo = s_m[wave][n], both = fmaxf(m[t], mo), base = both == -INFINITY ? 0.f : both;
          const float x = exp2_of(m[t] - base), y = exp2_of(mo - base);
          m[t] = both;
          l[t] = l[t] * x + s_l[wave][n] * y;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[t][i] = o[t][i] * x + s_o[wave][i][lane] * y;
        }
      }
      if (wave == 0 && r[t].real) put_row<T, D>(a, r[t], split, g, m[t], l[t], o[t]);
    }
    __syncthreads();
  }
  if constexpr (FEW) step_mass<T, FMT, D>(a, w, e, head, rows, start, 0, 1, s_lse);      // what the workgroup left in memory is there since the barrier
}

// Prompts: one workgroup, 128 query rows of a kv head.  Every step's blocks of keys and values (16 KB of codes, 32 KB as operands) are widened once, an equal share by
// every wave, into one of two buffers of shared memory, while the other is read: a code is widened once for 128 rows and not for 32, and no states are joined at
// the end.  Operands lie in shared memory as the lanes read them, 16 bytes a lane, without bank conflicts.  Four waves of 32 rows read least (D <= 128: 224 registers);
// heads of 256 take eight waves of 16 rows, whose outputs and queries fit beside the rest.  8000 rows of 32 / 8 heads of 128 over themselves: 500 us, 1.05 PFLOP/s; bound
// by shared memory's reads (one for two products) and, for few tiles, by those that have a compute unit to themselves (1.5 us a step, two together 1.0 each).
template <int D> constexpr int prompt_blocks() { return 512 / D; }   // of a step
template <int D> constexpr int prompt_tiles() { return D == 256 ? 1 : 2; }   // of sixteen rows, a wave

template <int FMT, int D>
__global__ __launch_bounds__(64 * 8 / prompt_tiles<D>(), 2) void kv8_prompt_kernel(AttnArgs a) {
  typedef uint16_t T;
  constexpr int C = D / 64, KB = prompt_blocks<D>(), NT = prompt_tiles<D>();
  // a step is 8 units of keys (a block's 64 values) and 4 of values (a pair of blocks' 64): four waves take two and one, of eight the first four one of values, the others two of keys
  constexpr bool kRoles = NT == 1;
  constexpr int kSets = D == 256 ? 2 : 1;   // steps of codes on their way to the registers
  constexpr bool kScaled = FMT == kE4m3;
  // keys [block][chunk][half], then values [pair of blocks][chunk][value of the lane's four]
  __shared__ bf16x8_t s_kv[2][2 * KB * C + 2 * KB * C][64];
  const int e = (blockIdx.y + blockIdx.z / a.n_split / a.round) % gridDim.y, head = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  const int len = start + rows.n, n_tiles = (total + kPromptRows - 1) / kPromptRows, split = blockIdx.z % a.n_split, stride = gridDim.z / a.n_split;
  for (int at = blockIdx.z / a.n_split; at < n_tiles; at += stride) {
    const int tile = a.snake && at >= a.round ? at - a.round : n_tiles - 1 - at;     // the rows that see most first
    QueryRow r[NT];
    bf16x8_t qf[NT][C][2];
    float m[NT], l[NT];
    f32x4 o[NT][D / 16];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      r[t] = query_row(tile * kPromptRows + (wave * NT + t) * 16 + n, total, a.group, rows, start, head);
      const T* qp = static_cast<const T*>(a.q) + r[t].row * a.q_stride + (int64_t)r[t].head * D + g * 16;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        kv8_query(qp + c * 64, &qf[t][c][0]);
        kv8_query(qp + c * 64 + 8, &qf[t][c][1]);
      }
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int all_see = tile * kPromptRows / a.group + start, any_sees = min((tile + 1) * kPromptRows - 1, total - 1) / a.group + start;
    const int blocks = min(any_sees / kKv8Page + 1, a.c.blocks(e)), per = (max(a.split_blocks, (blocks + a.n_split - 1) / a.n_split) + KB - 1) / KB * KB;
    const int b_lo = split * per, b_hi = min(blocks, b_lo + per);
    auto lane_of = [](float v, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
    for (int run = b_lo; run < b_hi; run += 64) {
      const int pid = run + lane < b_hi ? a.c.page(e, run + lane) : -1;
      const float ks = pid < 0 ? 0.f : *a.c.scale(pid, 0, head), vs = pid < 0 ? 0.f : *a.c.scale(pid, 1, head);
      const uint64_t there = __builtin_amdgcn_ballot_w64(pid >= 0);
      const int steps = (min(b_hi - run, 64) + KB - 1) / KB;
      const bool keys = !kRoles || wave >= 4, values = !kRoles || wave < 4;
      const int k_unit = (kRoles ? wave - 4 : wave) * 2, v_unit = wave;
      u32x4 kw[kSets][2], vw[kSets][2];    // of a set: two units of keys; the two blocks of a unit of values
      auto load = [&](int i, auto set) {
        if (i >= steps) return;
        if (keys)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int h = (k_unit + u) / C, c = (k_unit + u) % C;
            const int page = max(__builtin_amdgcn_readlane(pid, i * KB + h), 0);     // one that is not there: page 0's bytes, masked below
            kw[set()][u] = *reinterpret_cast<const u32x4*>(a.c.block(page, 0, head, D) + c * 1024 + n * 64 + g * 16);
          }
        if (values)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int h = v_unit / C * 2 + u, c = v_unit % C;
            const int page = max(__builtin_amdgcn_readlane(pid, i * KB + h), 0);
            vw[set()][u] = *reinterpret_cast<const u32x4*>(a.c.block(page, 1, head, D) + c * 1024 + g * 256 + n * 16);
          }
      };
      auto widen = [&](int i, auto set) {
        if (i >= steps) return;
        bf16x8_t (*to)[64] = s_kv[i & 1];
        u32x4 (&k)[2] = kw[set()], (&v)[2] = vw[set()];
        if (keys)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int unit = k_unit + u;
            const float x = lane_of(ks, i * KB + unit / C);
            to[unit * 2][lane] = kv8_operand<FMT>(k[u].x, k[u].y, x);
            to[unit * 2 + 1][lane] = kv8_operand<FMT>(k[u].z, k[u].w, x);
          }
        if (values) {
          const int h = v_unit / C * 2;
          const uint64_t want = ((1ull << KB) - 1) << (i * KB);
          if ((run + (i + 1) * KB) * kKv8Page > len || (there & want) != want) {
            // what lies behind the entry's last token may be any bytes, and 0 times one of them a NaN
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int here = there >> (i * KB + h + u) & 1 ? len - ((run + i * KB + h + u) * kKv8Page + 4 * g) : 0;
              v[u] &= here >= 4 ? 0xFFFFFFFFu : here <= 0 ? 0u : 0xFFFFFFFFu >> (32 - 8 * here);
            }
          }
          const float x = lane_of(vs, i * KB + h), y = lane_of(vs, i * KB + h + 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) to[2 * KB * C + v_unit * 4 + j][lane] = kv8_operand2<FMT>(v[0][j], v[1][j], x, y);
        }
      };
      constexpr std::integral_constant<int, 0> s0{};
      constexpr std::integral_constant<int, kSets - 1> s1{};
      load(0, s0);
      if (kSets == 2) load(1, s1);
      __syncthreads();                     // the run before has read its last buffer
      widen(0, s0);
      load(kSets, s0);
      auto body = [&](int i, auto set) {   // set: holds step i + 1
        __syncthreads();
        bf16x8_t (*from)[64] = s_kv[i & 1];
        const int slot0 = (run + i * KB) * kKv8Page;
        f32x4 s[NT][KB];
#pragma unroll
        for (int h = 0; h < KB; ++h)
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < KB; ++h) {
              const bf16x8_t kf = from[(h * C + c) * 2 + k][lane];
#pragma unroll
              for (int t = 0; t < NT; ++t) s[t][h] = mfma16(kf, qf[t][c][k], s[t][h]);
            }
        widen(i + 1, set);
        load(i + 1 + kSets, set);
        settle<NT, KB>(s);
        float f[KB];                       // the scores are scaled as they enter the exponential, but for masked steps: infinity times a factor that underflows is no mask
#pragma unroll
        for (int h = 0; h < KB; ++h) f[h] = kScaled ? a.scale_log2 : lane_of(ks, i * KB + h) * a.scale_log2;
        const uint64_t want = ((1ull << KB) - 1) << (i * KB);
        if (slot0 + KB * kKv8Page - 1 > all_see || (there & want) != want) {
#pragma unroll
          for (int h = 0; h < KB; ++h) {
            const int end = there >> (i * KB + h) & 1 ? INT32_MAX : -1, at0 = slot0 + h * kKv8Page + 4 * g;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[t][h][j] = at0 + j <= min(r[t].far, end) ? s[t][h][j] * f[h] : -INFINITY;
            f[h] = 1.f;
          }
        }
        bf16x8_t pf[NT][KB / 2];
        float top[NT];
        bool moves = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          top[t] = -INFINITY;
#pragma unroll
          for (int h = 0; h < KB; ++h) {
            if constexpr (kScaled) top[t] = max3(max3(top[t], s[t][h][0], s[t][h][1]), s[t][h][2], s[t][h][3]);
            else top[t] = fmaxf(top[t], max3(max3(s[t][h][0], s[t][h][1], s[t][h][2]), s[t][h][3], s[t][h][3]) * f[h]);
          }
          if constexpr (kScaled) top[t] *= f[0];      // one factor for all: the conversion took the blocks' scales along
          moves |= top[t] > m[t] + kSlack;
        }
        if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const float mx = quad_max(top[t]), to = mx > m[t] + kSlack ? mx : m[t], alpha = to == -INFINITY ? 1.f : exp2_of(m[t] - to);
            m[t] = to;
            l[t] *= alpha;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) o[t][d] *= alpha;
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float base = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
          for (int h = 0; h < KB; h += 2) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              p[j] = exp2_of(fmaf(s[t][h + j / 4][j & 3], f[h + j / 4], -base));
              l[t] += p[j];
              if (!kScaled) p[j] *= lane_of(vs, i * KB + h + j / 4);
            }
            kv8_split<1>(p, &pf[t][h / 2]);
          }
        }
#pragma unroll
        for (int h = 0; h < KB; h += 2)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bf16x8_t vf = from[2 * KB * C + (h / 2 * C + c) * 4 + j][lane];
#pragma unroll
              for (int t = 0; t < NT; ++t) o[t][4 * c + j] = mfma16(vf, pf[t][h / 2], o[t][4 * c + j]);
            }
      };
      for (int i = 0; i < steps; i += 2) {
        body(i, s1);
        if (i + 1 < steps) body(i + 1, s0);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] = quad_sum(l[t]);
      if (r[t].real) put_row<T, D>(a, r[t], split, g, m[t], l[t], o[t]);
    }
  }
}

// The splits' states of a (row, head) into its output: a workgroup takes 64 of its values, a wave every W-th split, sixteen of them on their way at a time.  A launch
// and two memory round trips: 128 splits of 16 rows of 256 values 5 us.
template <typename T, int D>
__global__ __launch_bounds__(512) void kv8_merge_kernel(AttnArgs a) {
  constexpr int C = D / 64;
  __shared__ float s_o[8][64], s_l[8];
  const int e = blockIdx.z, head = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63, c = blockIdx.x % C;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  for (int rr = blockIdx.x / C; rr < total; rr += gridDim.x / C) {
    const QueryRow r = query_row(rr, total, a.group, rows, start, head);
    const int64_t rh = (int64_t)r.row * a.heads + r.head;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + rh * a.n_split;
    const float* part = a.part_o + rh * a.n_split * D + c * 64 + lane;
    float m = -INFINITY;
    for (int i = lane; i < a.n_split; i += 64) m = fmaxf(m, ml[i].x);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
    for (int at = wave; at < a.n_split; at += 16 * waves) {
      float p[16];
      f32x2 x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int z = min(at + i * waves, a.n_split - 1);
        p[i] = part[(int64_t)z * D];
        x[i] = ml[z];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // a split without a key left no sums: what is in their place is not looked at
        const bool some = at + i * waves < a.n_split && (x[i].y > 0.f || x[i].y != x[i].y);
        const float w = exp2_of(x[i].x - base);
        l += some ? x[i].y * w : 0.f;
        o += some ? p[i] * w : 0.f;
      }
    }
    if (lane == 0) s_l[wave] = l;
    s_o[wave][lane] = o;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < waves; ++w) {
        l += s_l[w];
        o += s_o[w][lane];
      }
      const bool some = l > 0.f || l != l;
      st(static_cast<T*>(a.out) + r.row * a.out_stride + (int64_t)r.head * D + c * 64 + lane, some ? o / l : 0.f);
      if (a.lse && lane == 0 && c == 0) a.lse[rh] = some ? m + __log2f(l) : INFINITY;
    }
    __syncthreads();
  }
}

// The same for many rows: a wave each, eight splits on their way at a time.
template <typename T, int D>
__device__ __forceinline__ void merge_row(const AttnArgs& a, const QueryRow& r, int lane) {
  constexpr int V = D / 64, N = 8;
  const int64_t rh = (int64_t)r.row * a.heads + r.head;
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + rh * a.n_split;
  const float* part = a.part_o + rh * a.n_split * D + lane * V;
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = 0.f;
  for (int z0 = 0; z0 < a.n_split; z0 += N) {
    f32x2 x[N];
    float p[N][V], to = m;
#pragma unroll
    for (int z = 0; z < N; ++z) {
      const int at = min(z0 + z, a.n_split - 1);
      x[z] = ml[at];
#pragma unroll
      for (int v = 0; v < V; ++v) p[z][v] = part[(int64_t)at * D + v];
      to = fmaxf(to, x[z].x);
    }
    const float base = to == -INFINITY ? 0.f : to, by = exp2_of(m - base);
    m = to;
    l *= by;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] *= by;
#pragma unroll
    for (int z = 0; z < N; ++z) {
      // a split without a key left no sums: what is in their place is not looked at
      const bool some = z0 + z < a.n_split && (x[z].y > 0.f || x[z].y != x[z].y);
      const float w = exp2_of(x[z].x - base);
      l += some ? x[z].y * w : 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] += some ? p[z][v] * w : 0.f;
    }
  }
  const bool some = l > 0.f || l != l;
  const float inv = some ? 1.f / l : 0.f;
  T* op = static_cast<T*>(a.out) + r.row * a.out_stride + (int64_t)r.head * D + lane * V;
  if constexpr (V == 1) st(op, o[0] * inv);
  else
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const float y[2] = {o[v] * inv, o[v + 1] * inv};
      st2(op + v, y);
    }
  if (a.lse && lane == 0) a.lse[rh] = some ? m + __log2f(l) : INFINITY;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_merge_rows_kernel(AttnArgs a) {
  const int e = blockIdx.z, head = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  for (int rr = blockIdx.x * 4 + wave; rr < total; rr += gridDim.x * 4) merge_row<T, D>(a, query_row(rr, total, a.group, rows, start, head), lane);
}

// The weights that a call gives to the cached tokens, from the sums that the attention left.  A wave holds four blocks of keys (two of 256 values) as operands while the workgroup walks
// the rows that see them, MT tiles of sixteen a step, which its four waves (each with keys of its own) fetch together, two steps ahead, into shared memory: a
// token's sum is one wave's, in the rows' order.  n_slice > 1, where that leaves too few workgroups: every slice of the rows leaves its sums in part,
// kv8_mass_sum_kernel adds them in order.  Bound by shared memory's reads (one for four products, of 256 values for two) and the exponentials: 8000 rows of 32 / 8 heads of
// 128 over themselves 350 us, 0.75 PFLOP/s of the scores; 3 prompts of up to 2000 of 16 / 4 x 256: 72.
template <int D> constexpr int mass_blocks() { return D == 256 ? 2 : 4; }   // of keys, a wave
template <typename T, int D> constexpr int mass_tiles() { return sizeof(T) == 2 ? 2 : 1; }   // fp32: three parts of every query

template <typename T, int FMT, int D>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? 2 : 1)) void kv8_mass_kernel(AttnArgs a, MassArgs w) {
  constexpr int NP = kv8_parts<T>(), C = D / 64, MB = mass_blocks<D>(), MT = mass_tiles<T, D>(), F = 2 * C * MT / 4;      // F: operands (a tile's rows, 32 values) a wave fetches
  static_assert(F >= 1 || MT == 1, "an operand a wave at least");
  __shared__ bf16x8_t s_q[2][2 * C * MT][NP][64];
  const int e = (blockIdx.y + blockIdx.z / w.n_slice) % gridDim.y, head = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  const int blocks = min((start + rows.n + kKv8Page - 1) / kKv8Page, a.c.blocks(e)), slice = blockIdx.z % w.n_slice, tiles = (total + 15) / 16;
  for (int w0 = blockIdx.z / w.n_slice * 4 * MB; w0 < blocks; w0 += gridDim.z / w.n_slice * 4 * MB) {
    const int b0 = w0 + wave * MB;
    int page[MB];
    float ks[MB];
    bf16x8_t kf[MB][C][2];
    u32x4 kw[MB][C];
#pragma unroll
    for (int h = 0; h < MB; ++h) page[h] = b0 + h < blocks ? a.c.page(e, b0 + h) : -1;
#pragma unroll
    for (int h = 0; h < MB; ++h) {
      const uint8_t* kb = a.c.block(max(page[h], 0), 0, head, D) + n * 64 + g * 16;      // one that is not there: page 0's bytes, whose sums are left out
#pragma unroll
      for (int c = 0; c < C; ++c) kw[h][c] = *reinterpret_cast<const u32x4*>(kb + c * 1024);
      ks[h] = *a.c.scale(max(page[h], 0), 0, head) * a.scale_log2;
    }
    f32x4 sum[MB];
#pragma unroll
    for (int h = 0; h < MB; ++h) sum[h] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int slot0 = b0 * kKv8Page, first = (int)((int64_t)max(w0 * kKv8Page - start, 0) * a.group / (16 * MT));   // the first step with a row that sees one of the workgroup's blocks
    const int steps = (tiles + MT - 1) / MT, per = (steps - first + w.n_slice - 1) / w.n_slice, from = first + slice * per, to = min(steps, from + per);
    // operand f of a step: tile f / (2 C), values 32 (f % (2 C)); wave w fetches f = w F .. (heads of 64 in fp32: the first two waves one each)
    T raw[2][F > 0 ? F : 1][8] __attribute__((aligned(16)));
    float lse[2][MT];
    constexpr int FW = F > 0 ? F : 1;
    const bool fetches = F > 0 || wave < 2 * C * MT;
    auto fetch = [&](int step, auto set) {
      if (fetches && step < to)
#pragma unroll
        for (int f = 0; f < FW; ++f) {
          const int x = wave * FW + f, t = x / (2 * C), c = x % (2 * C) / 2, k = x & 1;
          const QueryRow r = query_row((step * MT + t) * 16 + n, total, a.group, rows, start, head);
          __builtin_memcpy(raw[set()][f], __builtin_assume_aligned(static_cast<const T*>(a.q) + r.row * a.q_stride + (int64_t)r.head * D + g * 16 + c * 64 + 8 * k, 16), 8 * sizeof(T));
        }
    };
    auto leave = [&](int step, auto set) {
      if (fetches && step < to)
#pragma unroll
        for (int f = 0; f < FW; ++f) {
          bf16x8_t q[NP];
          kv8_query(raw[set()][f], q);
#pragma unroll
          for (int p = 0; p < NP; ++p) s_q[(step - from) & 1][wave * FW + f][p][lane] = q[p];
        }
    };
    auto sums_of = [&](int step, auto set) {
      if (step < to)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const QueryRow r = query_row((step * MT + t) * 16 + n, total, a.group, rows, start, head);
          const float x = a.lse[(int64_t)r.row * a.heads + r.head];
          lse[set()][t] = r.real ? x : INFINITY;                     // a row behind the last weighs nothing
        }
    };
    constexpr std::integral_constant<int, 0> s0{};
    constexpr std::integral_constant<int, 1> s1{};
#pragma unroll
    for (int h = 0; h < MB; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        kf[h][c][0] = kv8_operand<FMT>(kw[h][c].x, kw[h][c].y);
        kf[h][c][1] = kv8_operand<FMT>(kw[h][c].z, kw[h][c].w);
        __builtin_amdgcn_sched_barrier(0);                 // one after the other, and before the queries take registers: all floats of the keys at once spill
      }
    fetch(from, s0);
    sums_of(from, s0);
    fetch(from + 1, s1);
    sums_of(from + 1, s1);
    __syncthreads();                                       // the blocks before have read their last buffer
    leave(from, s0);
    fetch(from + 2, s0);
    auto body = [&](int step, auto set, auto other) {      // set: holds the step's sums, other: the next step's queries
      const int buffer = (step - from) & 1;
      __syncthreads();
      f32x4 s[MT][MB];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < MB; ++h) s[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) {
              const bf16x8_t q = s_q[buffer][(t * C + c) * 2 + k][p][lane];
#pragma unroll
              for (int h = 0; h < MB; ++h) s[t][h] = mfma16(kf[h][c][k], q, s[t][h]);
            }
      leave(step + 1, other);
      fetch(step + 3, other);
      const bool all = slot0 + MB * kKv8Page - 1 <= step * MT * 16 / a.group + start;           // every row of the step sees every slot
      if (all) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int h = 0; h < MB; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[h][i] += exp2_of(fmaf(s[t][h][i], ks[h], -lse[set()][t]));
      } else {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int far = query_row((step * MT + t) * 16 + n, total, a.group, rows, start, head).far;
#pragma unroll
          for (int h = 0; h < MB; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[h][i] += slot0 + h * kKv8Page + 4 * g + i <= far ? exp2_of(fmaf(s[t][h][i], ks[h], -lse[set()][t])) : 0.f;
        }
      }
      sums_of(step + 2, set);
    };
    for (int step = from; step < to; step += 2) {
      body(step, s0, s1);
      if (step + 1 < to) body(step + 1, s1, s0);
    }
#pragma unroll
    for (int h = 0; h < MB; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = row16_sum(sum[h][i]);
        const int t = 4 * g + i, at = head * kKv8Page + t;
        if (n != i || page[h] < 0 || slot0 + h * kKv8Page + t >= start + rows.n) continue;
        if (w.n_slice > 1) w.part[((int64_t)slice * a.c.n_ids + a.c.indptr[e] + b0 + h) * a.c.kv_heads * kKv8Page + at] = x;
        else put_mass(w, page[h], at, x);
      }
  }
}

// The weights of steps over many tokens.  Where the keys were split, the first `merges` workgroups of an entry and head join its outputs and the others take the rows'
// log-sums from the splits' states: one launch for both (16 x 4096 tokens: 29.7 -> 27.5 us).
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256, (D == 128 ? 7 : 6)) void kv8_step_finish_kernel(AttnArgs a, MassArgs w, int merges) {
  __shared__ float s_lse[kStepRows];
  const int e = blockIdx.y, head = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e], total = rows.n * a.group;
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  if ((int)blockIdx.z < merges) {
    for (int rr = blockIdx.z * 4 + wave; rr < total; rr += merges * 4) merge_row<T, D>(a, query_row(rr, total, a.group, rows, start, head), lane);
    return;
  }
  step_mass<T, FMT, D>(a, w, e, head, rows, start, blockIdx.z - merges, gridDim.z - merges, s_lse);
}

// the slices' sums of a block's tokens, in order: a wave four blocks of a head
__global__ __launch_bounds__(256) void kv8_mass_sum_kernel(AttnArgs a, MassArgs w) {
  const int e = blockIdx.z, head = blockIdx.y;
  const RowSpan rows = row_span(a.row0, e, a.n_rows);
  const int start = a.starts[e];
  if (rows.n == 0 || start < 0 || start > INT32_MAX - 2048 - rows.n) return;
  const int len = a.c.tokens(e, start + rows.n);
  for (int slot = blockIdx.x * 256 + threadIdx.x; slot < len; slot += gridDim.x * 256) {
    const int block = slot / kKv8Page, page = a.c.page(e, block), at = head * kKv8Page + slot % kKv8Page;
    if (page < 0) continue;
    float x = 0.f;
    for (int z = 0; z < w.n_slice; ++z) x += w.part[((int64_t)z * a.c.n_ids + a.c.indptr[e] + block) * a.c.kv_heads * kKv8Page + at];
    put_mass(w, page, at, x);
  }
}

constexpr int kWholeBlocks = PEGAINFER_KV8_WHOLE / kKv8Page;

// How a call is cut: rows of a workgroup, splits of the keys and slices of the weights' rows where those leave too few workgroups.
struct AttnPlan { bool prompt, few; int tiles, row_tiles, n_split, split_blocks, mass_groups, n_slice, score_rows, round, snake; };
inline int rows_hint(int max_rows, int n_rows) { return std::min(std::max(max_rows, 1), n_rows); }
inline AttnPlan attn_plan(const pegainfer_kv8_cache* cache, int n_rows, int max_rows, int max_len, int heads, int dtype) {
  AttnPlan p;
  const int64_t rows = (int64_t)rows_hint(max_rows, n_rows) * (heads / cache->kv_heads), pairs = (int64_t)cache->kv_heads * cache->n_entries;
  p.row_tiles = rows > 16 && !(dtype == kDtF32 && cache->dim == 256) ? 2 : 1;
  p.prompt = dtype == kDtBf16 && rows >= kPromptRows;
  p.tiles = ceil_div(rows, p.prompt ? kPromptRows : 16 * p.row_tiles);
  const int blocks = std::max(1, ceil_div(max_len, kKv8Page));
  const int64_t want = 2 * device_cus();
  auto cut = [&](int64_t groups, int64_t most) { return (int)std::max<int64_t>(1, std::min((want + groups - 1) / groups, most)); };
  const int64_t groups = p.tiles * pairs;
  // Whole over a run of 64 blocks.  Steps over 1024 tokens of 8 heads of 128, called one by one: one entry 11.2 us whole, 13.5 cut with a merge, whose launch and workspace are
  // the host's; 32 entries 14.5 and 18.  Captured the cut is faster for few entries (11.1 and 8.5; 16 entries 13.2 and 11.6; 32 14.5 and 17.9).  Steps over more: runs of 16 blocks
  // at least.
  // Prompts: cut where they leave compute units without one (8 entries of 64 rows over 4000 tokens: 52 us in four, 64 in two), into runs of 32 blocks at least; a
  // split of 128 rows leaves 1 KB of sums a value of the head (32 entries of 32 rows over 1000 tokens, a workgroup a compute unit: 34 us whole, 46 halved).
  p.n_split = blocks <= kWholeBlocks ? 1
              : !p.prompt            ? cut(groups, std::min((blocks + 15) / 16, 256))
              : groups >= device_cus() ? 1
                                       : (int)std::max<int64_t>(1, std::min<int64_t>({want / groups, blocks / 32, 256}));
  p.split_blocks = ceil_div(blocks, p.n_split);
  p.few = blocks <= 32;                    // a step's weights by the attention's workgroups: two tokens a thread (500 tokens: 12.1 -> 11.8 us captured, 1024: 16.4 -> 17.9)
  p.round = (int)std::max<int64_t>(1, device_cus() / pairs);
  p.snake = p.n_split == 1 && p.tiles > p.round && p.tiles <= 2 * p.round;
  p.score_rows = rows <= kStepRows ? (int)rows : 0;
  p.mass_groups = p.score_rows ? ceil_div(blocks, 256 / kKv8Page) : ceil_div(blocks, 4 * (cache->dim == 256 ? mass_blocks<256>() : mass_blocks<128>()));
  // Weights: the first keys' rows are twice the average's.  Slices of 128 rows (four steps) at least: a step waits for its rows, 1 us, and the sum of the slices is a launch of 5
  // (88 tokens of 8 heads a group: 39 us whole, 26 in slices of 256, 22 of 128, 20 of 64; 30 rows over 4 x 2000 tokens 35, 35, 35, 36.5).
  p.n_slice = p.score_rows ? 1 : cut((p.mass_groups * pairs + 1) / 2, std::min<int64_t>((rows + 127) / 128, 16));
  return p;
}
// workgroups of `items` pieces of work cut `ways`, in whole pieces; kernels walk what a grid cannot hold
inline int deal(int64_t items, int ways) { return (int)std::min<int64_t>(items, 65000 / ways) * ways; }
// the splits' sums and states of a workspace, up to 16 bytes
inline int64_t split_floats(const AttnPlan& p, int64_t row_heads, int dim) { return p.n_split > 1 ? (row_heads * p.n_split * (dim + 2) + 3) / 4 * 4 : 0; }

}  // namespace pk

using namespace pk;

extern "C" {

int64_t pegainfer_kv8_attention_workspace(const pegainfer_kv8_cache* cache, int32_t n_rows, int32_t max_rows, int32_t max_len, int32_t heads, int32_t dtype,
                                          int32_t with_mass) {
  if (!kv8_ok(cache) || n_rows <= 0 || max_rows < 0 || max_len < 0 || heads < cache->kv_heads || cache->n_entries == 0) return 0;
  const AttnPlan p = attn_plan(cache, n_rows, max_rows, max_len, heads, dtype);
  const int64_t rh = (int64_t)n_rows * heads;
  const int64_t slots = (int64_t)cache->n_page_ids * cache->kv_heads * kKv8Page;
  return split_floats(p, rh, cache->dim) +
         (with_mass ? (rh + 3) / 4 * 4 + (p.n_slice > 1 ? p.n_slice * slots : 0) + p.score_rows * slots : 0);
}

pegainfer_status_t pegainfer_kv8_attention(const pegainfer_kv8_cache* cache, const pegainfer_kv8_attn_desc* d, pegainfer_stream_t stream) {
  if (!kv8_ok(cache) || !d || (d->dtype != kDtBf16 && d->dtype != kDtF32) || d->heads < 1 || d->heads % cache->kv_heads || d->n_rows < 0 || d->max_rows < 0 || d->max_len < 0 ||
      !(d->scale >= 0.f))
    return PK_BAD;
  if (d->n_rows == 0 || cache->n_entries == 0) return 0;
  const int64_t width = (int64_t)d->heads * cache->dim, unit = d->dtype == kDtBf16 ? 8 : 4;
  if (!d->q || !d->out || !d->row0 || !d->starts || !host_aligned16(d->q) || !host_aligned16(d->out) || d->q_row_stride < width || d->out_row_stride < width ||
      d->q_row_stride % unit || d->out_row_stride % unit || (int64_t)d->n_rows * (d->heads / cache->kv_heads) > INT32_MAX - 1024)
    return PK_BAD;
  const bool weigh = d->mass_out != nullptr;
  const int64_t mass_width = (int64_t)cache->kv_heads * kKv8Page;
  if (weigh && (d->mass_out_page_stride < mass_width || (d->mass_keep != 0.f && (!d->mass || d->mass_page_stride < mass_width)))) return PK_BAD;
  const int group = d->heads / cache->kv_heads;
  const AttnPlan p = attn_plan(cache, d->n_rows, d->max_rows, d->max_len, d->heads, d->dtype);
  if ((weigh || p.n_split > 1) && (!d->workspace || !host_aligned16(d->workspace))) return PK_BAD;
  const int64_t rh = (int64_t)d->n_rows * d->heads;
  // workspace: the splits' sums and states, the rows' log-sums, then either the slices' sums or the scores (never both: those are of few rows)
  float* const part_ml = p.n_split > 1 ? d->workspace + rh * p.n_split * cache->dim : nullptr;
  float* const lse = weigh ? d->workspace + split_floats(p, rh, cache->dim) : nullptr;
  float* const rest = weigh ? lse + (rh + 3) / 4 * 4 : nullptr;
  const AttnArgs a{kv8_of(cache), d->q, d->q_row_stride, d->out_row_stride, d->row0, d->starts, d->n_rows, group, d->heads, p.n_split, p.split_blocks,
                   d->scale * 1.4426950408889634f, d->out, lse, d->workspace, part_ml, p.score_rows ? rest : nullptr, p.score_rows,
                   p.round, p.snake};
  // Grid (head, entry, work), the longest work first: heads next to one another meet their cache in their XCD's second level (8 heads: one each), and
  // the short ones fill the end.  The entries change places from round to round, and where two rounds are all the second starts with the shortest: what shares a
  // compute unit is a long piece and a short one.
  const dim3 grid(cache->kv_heads, cache->n_entries, deal(p.tiles, p.n_split)), mass_grid(cache->kv_heads, cache->n_entries, deal(p.mass_groups, p.n_slice));
  // splits of 2048 rows and heads fill the chip with a wave each; of fewer, a workgroup each shortens the walk over many splits
  const bool many = p.n_split <= 8 || rh >= 2048;
  const int64_t rows = (int64_t)rows_hint(d->max_rows, d->n_rows) * group;
  const dim3 merge_grid((uint32_t)(rows * (cache->dim / 64)), cache->kv_heads, cache->n_entries);
  const dim3 rows_grid(ceil_div(rows, 4), cache->kv_heads, cache->n_entries);
  const dim3 sum_grid(std::max(1, ceil_div(d->max_len, 256)), cache->kv_heads, cache->n_entries);
  const MassArgs w{d->mass, d->mass_out, rest, d->mass_page_stride, d->mass_out_page_stride, d->mass_keep, p.n_slice};
  kv8_by(d->dtype, cache->format, cache->dim, [&](auto* t, auto fmt, auto dim) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int D = dim();
    if constexpr (sizeof(T) == 2) {
      if (p.prompt) kv8_prompt_kernel<fmt(), D><<<grid, 64 * 8 / prompt_tiles<D>(), 0, as_stream(stream)>>>(a);
    }
    if constexpr (sizeof(T) == 2 || D < 256) {
      if (!p.prompt && p.row_tiles == 2) kv8_attn_kernel<T, fmt(), D, 2, false, false><<<grid, 256, 0, as_stream(stream)>>>(a, w);
    }
    if (!p.prompt && p.row_tiles == 1) {
      if (p.score_rows && weigh && p.few) kv8_attn_kernel<T, fmt(), D, 1, true, true><<<grid, 256, 0, as_stream(stream)>>>(a, w);
      else if (p.score_rows) kv8_attn_kernel<T, fmt(), D, 1, true, false><<<grid, 256, 0, as_stream(stream)>>>(a, w);
      else if constexpr (sizeof(T) == 4 && D == 256) kv8_attn_kernel<T, fmt(), D, 1, false, false><<<grid, 256, 0, as_stream(stream)>>>(a, w);
    }
    const bool step = weigh && p.score_rows, merge = p.n_split > 1 && !step;
    if (merge && many) kv8_merge_rows_kernel<T, D><<<rows_grid, 256, 0, as_stream(stream)>>>(a);
    if (merge && !many) kv8_merge_kernel<T, D><<<merge_grid, 64 * std::min(8, p.n_split), 0, as_stream(stream)>>>(a);
    const int merges = p.n_split > 1 ? ceil_div(p.score_rows, 4) : 0;
    if (step && !p.few) kv8_step_finish_kernel<T, fmt(), D><<<dim3(mass_grid.x, mass_grid.y, mass_grid.z + merges), 256, 0, as_stream(stream)>>>(a, w, merges);
    if (weigh && !step) kv8_mass_kernel<T, fmt(), D><<<mass_grid, 256, 0, as_stream(stream)>>>(a, w);
  });
  if (weigh && p.n_slice > 1) kv8_mass_sum_kernel<<<sum_grid, 256, 0, as_stream(stream)>>>(a, w);
  return (pegainfer_status_t)hipGetLastError();
}

}  // extern "C"
