// Attention over a paged cache of 4 bits (cache4.h), for one head size (QRT_HEAD_DIM).
//
// Scores are formed transposed, S^T = K Q^T, and outputs O^T = V^T P^T, on the bfloat16 MFMA of 16 x 16 x 32. A code n is put under an
// exponent by a mask and an or, OFF + n exactly, two at a time, and what that adds is taken out again behind the sums:
//   score = step * (sum q (OFF + n)) + (lo - OFF step) * sum q
//   out   = sum w (OFF + n) + sum (p (lo + 8 step) - (OFF + 8) w),  w = p * step rounded as it is multiplied,
// so that w's rounding multiplies n - 8 alone. Keys and values of 16 keys are D / 8 neighbouring bytes a lane: no operand crosses
// lanes and nothing goes through LDS. A block of 32 keys is on its way while another is multiplied, its page numbers one block before that.
//
// bfloat16 queries: OFF = 128, weights w in bfloat16 (their errors average out, as in every attention that multiplies
// probabilities in 16 bits). float32 queries: q and w as three bfloat16 each (24 bits in all, whole), and OFF = -8, which leaves nothing to
// take out: with an offset of 16 the results were 3.6e-6 from those in 64 bits, where sums in float32 are 2e-7.
//
// A wave has 16 RT rows (token x head of the group) of its own. Of a block's four waves GROUPS share the same rows, take the blocks of keys in
// turn and meet in LDS at the end; the rows are 4 / GROUPS bands of 16 RT, whose waves read the same keys at about the same time. Many groups
// make many blocks of few rows, which fills the chip and evens out what a causal mask leaves; few groups meet less often. us with 4, 2 and
// 1 groups, 32 heads on 8 of 128, a prompt read at once: 300 tokens (304 blocks of 4 groups) 11.5, 12.1, 15.3; 512 (512) 12.8, 14.7, 21.3;
// 700 (704) 22.2, 19.4, 27.4; 2,048 (2,048) 67.7, 59.0, 70.3; two of 2,048 (4,096) 140, 119, 115.
// RT = 2 takes the codes out of their words half as often a row: from 384 blocks on, nearly as many as the chip holds, that is what counts (400 tokens
// of 4,096 49.6 and 60.1 us), before that the blocks are (128 tokens 8.7 and 5.9). A launch may cut the keys into pieces of one length as well,
// which a second kernel joins. Sums, maxima and outputs are float32.
//
// What bounds it: many rows, the vector instructions: some 276 a block of 32 keys and 32 rows beside 34 of the matrix cores, issued in 62 % of the
// cycles at 2,048 tokens (0.58 PFLOP/s). Taken out on the way there: a branch an element that the compiler had made of one condition
// (93 us -> 71), and arguments held in scalar registers, which it kept in a vector register's lanes (71 -> 64). One row a head over 32,000 tokens: 34.8 MB in
// some 11 us, 3.2 TB/s, eight blocks of keys a wave between a start of three trips to memory and a meeting, and a merge of 3.5 us; its waves wait in 41 %
// of their time with one block of keys on its way.
#include "common.h"
#include "cache4.h"

constexpr int D = QRT_HEAD_DIM;
static_assert(D % 32 == 0 && D >= 32 && D <= 256, "heads of 32 to 256 in steps of 32");
constexpr int KS = D / 32;  // steps of 32 elements: words a lane holds of 16 keys, and of 16 values
typedef float f32x2_t __attribute__((ext_vector_type(2)));
constexpr float LOG2E = 1.4426950408889634f;

// What follows from a step's lengths, the same for all its layers.
struct Attention4Plan {
  const int* tile_seq;      // null: tile i is sequence i from its first row
  const int* tile_row0;     // null: from the first row
  const int* merge_tokens;  // null: all
  int num_merge_tokens, num_tiles, nq, nkv;
  int window, chunk, keep_first;
  int piece, pieces;  // blocks of 32 keys in a piece; how many pieces the launch has room for
};
struct Attention4Args : Attention4Plan {
  const void* q;
  void* out;
  const uint8_t* k;
  const uint8_t* v;
  const unsigned* steps;
  const int* cu_q;
  const int* kv_lens;
  const int* table;
  float* part_o;   // [rows, pieces, D], not divided by the sums
  float* part_ml;  // [rows, pieces, 2]
  int table_width, num_pages, page_size, sink;
  float scale, softcap;
  PageMagic page, group;  // division by the page size, and by the query heads of a key head
};
#ifdef __HIP_DEVICE_COMPILE__
// The kernel's arguments, read where they are wanted: held from the start they took so many scalar registers that the loop over keys moved
// forty of them a block in and out of a vector register's lanes.
typedef const Attention4Args __attribute__((address_space(4)))* Arguments;
__device__ __forceinline__ Arguments arguments() {
  Arguments a = (Arguments)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}
#endif

// The blocks of 32 keys that rows [base, base + rows_of_tile) of a sequence see: first those of the kept first tokens, then a run.
struct Blocks {
  int kept, first, count;
  __device__ __forceinline__ int at(int i) const { return i < kept ? i : first + i - kept; }
};
__device__ __forceinline__ int lowest_seen(const Attention4Args& a, int pos) {
  if (a.window) return max(0, pos - a.window + 1);
  return a.chunk ? pos - pos % a.chunk : 0;
}
__device__ __forceinline__ int token_of_row(const Attention4Args& a, int row) {
  int token, in_group;
  page_of(a.group, row, token, in_group);
  return token;
}
__device__ __forceinline__ Blocks blocks_of(const Attention4Args& a, int base, int tile_rows, int rows, int before) {
  const int last = before + token_of_row(a, min(base + tile_rows, rows) - 1);
  const int low = lowest_seen(a, before + token_of_row(a, base));
  Blocks b;
  b.first = low >> 5;
  b.kept = min((a.keep_first + 31) >> 5, b.first);
  b.count = b.kept + (last >> 5) + 1 - b.first;
  return b;
}

template <int N>
struct Words {
  unsigned w[N];
};
template <int N>
__device__ __forceinline__ Words<N> load_words(const void* p) {
  Words<N> r;
  __builtin_memcpy(&r, __builtin_assume_aligned(p, N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4), sizeof(r));
  return r;
}

#ifdef __HIP_DEVICE_COMPILE__  // the host's compiler knows no buffer resources
template <int N>
__device__ __forceinline__ Words<N> load_words(const __amdgpu_buffer_rsrc_t from, unsigned lane_at, unsigned at) {
  Words<N> r;
  constexpr int FOURS = N / 4, REST = N % 4;
#pragma unroll
  for (int i = 0; i < FOURS; ++i) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b128(from, lane_at + 16 * i, at, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.w[4 * i + e] = x[e];
  }
  if constexpr (REST == 1) {
    r.w[N - 1] = __builtin_amdgcn_raw_buffer_load_b32(from, lane_at + 16 * FOURS, at, 0);
  } else if constexpr (REST == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(from, lane_at + 16 * FOURS, at, 0);
    r.w[N - 2] = x[0], r.w[N - 1] = x[1];
  } else if constexpr (REST == 3) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b96(from, lane_at + 16 * FOURS, at, 0);
    r.w[N - 3] = x[0], r.w[N - 2] = x[1], r.w[N - 1] = x[2];
  }
  return r;
}
#endif

struct Stage {
  Words<KS> k[2], v[2];
  unsigned s;  // lanes below 32: lo and step of key `lane`, the others: of value `lane` - 32
};
// What a lane makes of the pairs of its wave's 32 keys, one pair a lane, for all to read: of keys what multiplies a sum and a query's
// sum, of values the step and the middle.
struct Scales {
  float kmul[32], kadd[32], vstep[32], vmid[32];
};

// Nibbles `nibble` and `nibble` + 4 of x as a pair of bfloat16, OFF + n each. OFF = 128: mask and exponent are kept in registers where the
// compiler does not see their values: it then takes one instruction, v_and_or_b32, for what two with literals would do. OFF = -8: by way
// of float32, five instructions a pair for two.
template <int OFF>
struct Place;
template <>
struct Place<128> {
  unsigned mask, exponent;
  __device__ __forceinline__ Place() {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(mask));
    asm("v_mov_b32 %0, 0x43004300" : "=v"(exponent));
  }
  __device__ __forceinline__ unsigned operator()(unsigned x, int nibble) const { return ((x >> (4 * nibble)) & mask) | exponent; }
};
template <>
struct Place<-8> {
  __device__ __forceinline__ unsigned operator()(unsigned x, int nibble) const {
    const unsigned bytes = (nibble & 1 ? x >> 4 : x) & 0x0f0f0f0fu;
    const int at = 8 * (nibble >> 1);
    typedef bf16_t bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t pair = {(bf16_t)((float)(bytes >> at & 255u) - 8.f), (bf16_t)((float)(bytes >> (at + 16) & 255u) - 8.f)};
    return __builtin_bit_cast(unsigned, pair);
  }
};

constexpr float NOTHING = -3.4028235e38f;  // the reference of a row that has seen no key

template <int RT, int NS, bool CAP>
struct Walk {
  static constexpr int OFF = NS == 1 ? 128 : -8;
  Place<OFF> place;
  bf16x8_t q[NS][RT][KS];
  float qsum[RT];              // sum of the row's query, times the unit of the scores
  float ref[RT];               // what exponents are taken against, in log2
  float l[RT], c[RT];          // this lane's part of sum e, and of sum e (lo + 8 step)
  int pos[RT], low[RT];
  f32x4_t acc[RT][2 * KS], weights[RT];  // sum w (OFF + n) since the last time the offsets were taken out; sum w since then, four times the same

  template <typename T>
  __device__ __forceinline__ void load_queries(const Attention4Args& a, float unit, int head, PageMagic g, int q0, int base, int rows, int before, int lane) {
    const int quad = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = min(base + 16 * t + (lane & 15), rows - 1);
      int token, in_group;
      page_of(g, r, token, in_group);
      pos[t] = before + token;
      low[t] = lowest_seen(a, pos[t]);
      const T* src = (const T*)a.q + ((size_t)(q0 + token) * a.nq + head * (int)g.size + in_group) * D + quad * (D / 4);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float x[8];
        if constexpr (sizeof(T) == 2) {
          const bf16x8_t y = *(const bf16x8_t*)(src + 8 * s);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
        } else {
          const f32x4_t y = *(const f32x4_t*)(src + 8 * s), z = *(const f32x4_t*)(src + 8 * s + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = y[e], x[4 + e] = z[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += x[e];
          float rest = x[e];
#pragma unroll
          for (int n = 0; n < NS; ++n) {  // in the order in which codes leave their word: 0 and 4, 1 and 5, ...
            const bf16_t part = (bf16_t)rest;
            q[n][t][s][e < 4 ? 2 * e : 2 * (e - 4) + 1] = part;
            rest -= (float)part;
          }
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      qsum[t] = sum * unit;
      ref[t] = NOTHING, l[t] = 0.f, c[t] = 0.f;
      weights[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < 2 * KS; ++d) acc[t][d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
  }

  // One block of 32 keys. `inside`: every row of the wave sees all of it. `unit`: of the scores, log2 but with a cap.
  __device__ __forceinline__ void block(const Attention4Args& a, float unit, const Stage& st, Scales& scales, int b, bool inside, int lane) {
    const int quad = lane >> 4;
    const bool of_value = lane >= 32;
    {
      const float step = __uint_as_float(st.s & 0xffff0000u), lo = __uint_as_float(st.s << 16);
      float* to = (float*)&scales + (of_value ? 32 : 0) + lane;  // lane - 32 of the third array, or lane of the first
      to[0] = step * (of_value ? 1.f : unit);
      to[32] = fmaf(of_value ? 8.f : -(float)OFF, step, lo);
    }
    __builtin_amdgcn_wave_barrier();  // a wave's reads of LDS come behind its writes
    f32x4_t sc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) sc[t][h] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned x = st.k[h].w[s];
        const u32x4_t w = {place(x, 0), place(x, 1), place(x, 2), place(x, 3)};
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int n = 0; n < NS; ++n)
            sc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), q[n][t][s], sc[t][h], 0, 0, 0);
      }
    // of rows lane & 15 and keys 16 h + 4 quad + r: score = kmul * sc + kadd * qsum
    f32x4_t kmul[2], kadd[2], vstep[2], vmid[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kmul[h] = *(const f32x4_t*)(scales.kmul + 16 * h + 4 * quad), kadd[h] = *(const f32x4_t*)(scales.kadd + 16 * h + 4 * quad);
      vstep[h] = *(const f32x4_t*)(scales.vstep + 16 * h + 4 * quad), vmid[h] = *(const f32x4_t*)(scales.vmid + 16 * h + 4 * quad);
    }
    __builtin_amdgcn_wave_barrier();
    auto score = [&](int t, int h, int r) {
      const float x = fmaf(kmul[h][r], sc[t][h][r], kadd[h][r] * qsum[t]);
      return CAP ? a.softcap * tanhf(x / a.softcap) * LOG2E : x;
    };
    auto against = [&](int t, int h, int r) {  // the score less the reference
      return CAP ? score(t, h, r) - ref[t] : fmaf(kmul[h][r], sc[t][h][r], fmaf(kadd[h][r], qsum[t], -ref[t]));
    };
    // exponents against the reference, which moves only where a score is above it by more than 8
    float ex[RT][2][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) ex[t][h][r] = against(t, h, r);
    if (!inside) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = 32 * b + 16 * h + 4 * quad + r;
            const bool sees = (unsigned)(key - low[t]) <= (unsigned)(pos[t] - low[t]) || key < min(a.keep_first, pos[t] + 1);
            ex[t][h][r] = sees ? ex[t][h][r] : -INFINITY;
          }
    }
    bool above = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float top = fmaxf(fmaxf(fmaxf(ex[t][0][0], ex[t][0][1]), fmaxf(ex[t][0][2], ex[t][0][3])),
                              fmaxf(fmaxf(ex[t][1][0], ex[t][1][1]), fmaxf(ex[t][1][2], ex[t][1][3])));
      above |= top > 8.f;
    }
    if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float x = -INFINITY;  // the row's highest score, from all four quarters of its keys
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) x = fmaxf(x, ex[t][h][r] == -INFINITY ? -INFINITY : score(t, h, r));
        x = fmaxf(x, __shfl_xor(x, 16));
        x = fmaxf(x, __shfl_xor(x, 32));
        // by the row's own scores alone, whatever its neighbours need
        const float to = x - ref[t] > 8.f ? x : ref[t];
        const float by = to > ref[t] ? __builtin_amdgcn_exp2f(ref[t] - to) : 1.f;
        ref[t] = to;
        l[t] *= by, c[t] *= by;
        weights[t] *= by;
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) acc[t][d] *= by;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) ex[t][h][r] = ex[t][h][r] == -INFINITY ? -INFINITY : against(t, h, r);
      }
    }
    bf16x8_t p[NS][RT];
    if (inside) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = __builtin_amdgcn_exp2f(ex[t][h][r]);
            l[t] += e;
            c[t] = fmaf(e, vmid[h][r], c[t]);
            ex[t][h][r] = e * vstep[h][r];
          }
    } else {  // a value that is not finite touches only rows that see it
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool sees = ex[t][h][r] != -INFINITY;
            const float e = __builtin_amdgcn_exp2f(ex[t][h][r]);
            l[t] += e;
            c[t] = fmaf(e, sees ? vmid[h][r] : 0.f, c[t]);
            ex[t][h][r] = sees ? e * vstep[h][r] : 0.f;
          }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int slot = 4 * h + (r == 1 ? 2 : r == 2 ? 1 : r);  // codes leave a word of four tokens as 0 and 2, 1 and 3
          float rest = ex[t][h][r];
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            const bf16_t part = (bf16_t)rest;
            p[n][t][slot] = part;
            rest -= (float)part;
          }
        }
    constexpr unsigned ONES = 0x3f803f80u;
    const u32x4_t ones = {ONES, ONES, ONES, ONES};
    if constexpr (OFF != -8)
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < NS; ++n)
          weights[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ones), p[n][t], weights[t], 0, 0, 0);
#pragma unroll
    for (int w = 0; w < KS; ++w) {
      const unsigned x = st.v[0].w[w], y = st.v[1].w[w];
      const u32x4_t lo = {place(x, 0), place(x, 2), place(y, 0), place(y, 2)};
      const u32x4_t hi = {place(x, 1), place(x, 3), place(y, 1), place(y, 3)};
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          acc[t][2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, lo), p[n][t], acc[t][2 * w], 0, 0, 0);
          acc[t][2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, hi), p[n][t], acc[t][2 * w + 1], 0, 0, 0);
        }
    }
  }

  // The offsets of the codes out of the sums, which stay small so: what a sum of OFF w loses in its last places adds up over a long
  // walk to more than a flat softmax leaves of its values (32,000 keys: 0.8 % of them).
  __device__ __forceinline__ void center() {
    if constexpr (OFF == -8) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float off = -(float)(OFF + 8) * weights[t][0];
#pragma unroll
      for (int d = 0; d < 2 * KS; ++d) acc[t][d] += off;
      weights[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
  }

  // The lanes' parts together: of every row its sums, and what its outputs still lack.
  __device__ __forceinline__ void end() {
    center();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      l[t] += __shfl_xor(l[t], 16), l[t] += __shfl_xor(l[t], 32);
      c[t] += __shfl_xor(c[t], 16), c[t] += __shfl_xor(c[t], 32);
      if (ref[t] == NOTHING) ref[t] = -INFINITY;
    }
  }
};

template <typename T>
__device__ __forceinline__ void store_out4(T* to, f32x4_t x) {
  if constexpr (sizeof(T) == 4) *(f32x4_t*)to = x;
  else *(bf16x4_t*)to = (bf16x4_t){(bf16_t)x[0], (bf16_t)x[1], (bf16_t)x[2], (bf16_t)x[3]};
}
// What divides a row's sums: with a sink, one more term of score 0. `m` in log2, 0 for a row that sees nothing.
__device__ __forceinline__ float inverse_sum(float m, float l, bool sink) {
  if (sink) {
    if (m == -INFINITY) return 0.f;
    const float top = fmaxf(m, 0.f), by = __builtin_amdgcn_exp2f(m - top);
    return by / (l * by + __builtin_amdgcn_exp2f(-top));
  }
  return l == 0.f ? 0.f : 1.f / l;
}

// Waves a SIMD holds: one where queries and sums alone take most of half the registers, else two (three, of the kernels that could: level).
constexpr int residents(int RT, int NS) { return NS == 3 && D > 160 ? 1 : 2; }

// BY16: pages of a multiple of 16 tokens, so that 16 keys lie in one page and where they begin is the same for the whole wave, and pools of
// less than 4 GiB. A lane finds the page of 16 keys, 32 blocks of 32 at a time, and the loads take it from there into a scalar: finding
// pages with scalar instructions, block after block, took a hundred of them a block.
template <int RT, int NS, int GROUPS, int BANDS, bool CAP, bool BY16, typename T>
__global__ __launch_bounds__(64 * GROUPS * BANDS, residents(RT, NS)) void attention4_kernel(Attention4Args a) {
  const int lane = threadIdx.x & 63, wave = uniform_wave_number(), quad = lane >> 4;
  const int head = blockIdx.x, tile = blockIdx.y, piece = blockIdx.z;
  constexpr int TILE_ROWS = 16 * RT * BANDS;
  const int group = wave / BANDS, band = wave % BANDS;
  // What the launch's shapes hang on is read through the scalar cache: the page numbers of the first keys, which without a window do not
  // wait for the lengths, and these come together.
  typedef const int __attribute__((address_space(4)))* constant_ints;
  auto constant = [](const int* p, int i) { return ((constant_ints)p)[__builtin_amdgcn_readfirstlane(i)]; };
  const int seq = a.tile_seq ? constant(a.tile_seq, tile) : tile, row0 = a.tile_row0 ? constant(a.tile_row0, tile) : 0;
  const int g = a.group.size;
  const bool from_start = !a.window && !a.chunk;
  // A row: one token of a head. A page number from the table, wherever it points, is brought into the pool: given-back pages are
  // masked, but asked for.
  auto row_of_key = [&](const auto& a, int key) {
    int page, off;
    page_of(PageMagic{a.page.size, a.page.by}, key, page, off);
    const int entry = (a.table + (size_t)seq * a.table_width)[min(page, a.table_width - 1)];
    return (unsigned)((max(0, min(entry, a.num_pages - 1)) * a.nkv + head) * a.page_size + off);
  };
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int RAW = 0x00020000;  // a buffer of bytes
  const unsigned pool_rows = (unsigned)a.num_pages * a.nkv * a.page_size;
  const __amdgpu_buffer_rsrc_t k_buf = __builtin_amdgcn_make_buffer_rsrc((void*)a.k, 0, (int)(pool_rows * (D / 2)), RAW);
  const __amdgpu_buffer_rsrc_t v_buf = __builtin_amdgcn_make_buffer_rsrc((void*)a.v, 0, (int)(pool_rows * (D / 2)), RAW);
  const __amdgpu_buffer_rsrc_t s_buf = __builtin_amdgcn_make_buffer_rsrc((void*)a.steps, 0, (int)(pool_rows * 8), RAW);
#endif
  // keys 16 h + (lane & 15) and 16 h + 4 quad of block b; `found`: BY16, the rows that the lanes have found, those of this block in 2 j and 2 j + 1
  auto load = [&](int b, unsigned found, int j) {
    Stage st;
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (BY16) {
        const unsigned row = (unsigned)__builtin_amdgcn_readlane((int)found, 2 * j + h);
        st.k[h] = load_words<KS>(k_buf, (lane & 15) * (D / 2) + quad * (D / 8), row * (D / 2));
        st.v[h] = load_words<KS>(v_buf, quad * (2 * D) + (lane & 15) * (D / 8), row * (D / 2));
      } else {
        const size_t krow = row_of_key(a, 32 * b + 16 * h + (lane & 15)), grow = row_of_key(a, 32 * b + 16 * h + 4 * quad);
        st.k[h] = load_words<KS>(a.k + krow * (D / 2) + quad * (D / 8));
        st.v[h] = load_words<KS>(a.v + grow * (D / 2) + (lane & 15) * (D / 8));
      }
    }
    if constexpr (BY16) {
      const unsigned row0 = (unsigned)__builtin_amdgcn_readlane((int)found, 2 * j), row1 = (unsigned)__builtin_amdgcn_readlane((int)found, 2 * j + 1);
      st.s = load_words<1>(s_buf, 8 * ((lane & 16 ? row1 : row0) + (lane & 15)) + 4 * (lane >> 5), 0).w[0];
    } else {
      st.s = a.steps[2 * (size_t)row_of_key(a, 32 * b + (lane & 31)) + (lane >> 5)];
    }
#endif
    return st;
  };
  int i0 = piece * a.piece;
  constexpr int FOUND = 30;  // blocks of a batch: the lanes find 32, one of them is fetched in the batch before
  auto key_of_lane = [&](int b) { return 32 * b + 16 * (lane & 1); };
  unsigned found = 0;
  if (BY16 && from_start) found = row_of_key(a, key_of_lane(i0 + group + (lane >> 1) * GROUPS));
  const int q0 = constant(a.cu_q, seq), q_len = constant(a.cu_q, seq + 1) - q0, kv_len = constant(a.kv_lens, seq);
  const int rows = q_len * g, before = kv_len - q_len;
  if (row0 >= rows || before < 0) return;
  const Blocks all = blocks_of(a, row0, TILE_ROWS, rows, before);
  int end = min(all.count, i0 + a.piece);
  if (i0 >= all.count) {  // the sequence has no such piece: its parts say so
    for (int r = row0 + threadIdx.x; r < min(row0 + TILE_ROWS, rows); r += 64 * GROUPS * BANDS)
      *(f32x2_t*)(a.part_ml + 2 * (((size_t)(q0 + r / g) * a.nq + head * g + r % g) * a.pieces + piece)) = (f32x2_t){-INFINITY, 0.f};
    return;
  }
  const int base = row0 + band * 16 * RT;
  const int last_pos = before + token_of_row(a, min(base + 16 * RT, rows) - 1), first_pos = before + token_of_row(a, base);
  if (BANDS > 1) {
    if (GROUPS == 1 && base >= rows) return;
    // this wave's own rows may see less than the tile's
    end = base < rows ? min(end, all.kept + max(0, (last_pos >> 5) + 1 - all.first)) : 0;
    const int own_first = all.kept + (lowest_seen(a, first_pos) >> 5) - all.first;
    if (a.keep_first == 0) i0 = max(i0, own_first);
  }
  i0 += group;
  const int last_low = lowest_seen(a, last_pos);
  auto block_at = [&](int i) { return from_start ? i : all.at(max(0, min(i, all.count - 1))); };  // past the end none that is used
  Stage s0, s1;  // the first block is on its way while the queries are made ready
  if (i0 < end) {
    if (BY16 && !from_start) found = row_of_key(a, key_of_lane(block_at(i0 + (lane >> 1) * GROUPS)));
    s0 = load(block_at(i0), found, 0);
  }
  __shared__ __align__(16) Scales scales[GROUPS * BANDS];
  Walk<RT, NS, CAP> walk;
  const float unit = CAP ? a.scale : a.scale * LOG2E;
  walk.template load_queries<T>(a, unit, head, a.group, q0, base, rows, before, lane);

  auto use = [&](const Stage& st, int i) {
    const int b = block_at(i);
    const bool inside = 32 * b + 31 <= first_pos && (32 * b >= last_low || 32 * b + 31 < a.keep_first);
    walk.block(a, unit, st, scales[wave], b, inside, lane);
  };
  if (i0 < end) {
    unsigned later = 0;
    int j = FOUND;  // where the batch stands
    for (int i = i0;;) {
      if ((i - i0) / GROUPS % 8 == 0) walk.center();
      if (BY16 && j == FOUND) {  // j runs by two: a batch's rows are found while the one before is used
        if (i != i0) found = later;
#ifdef __HIP_DEVICE_COMPILE__
        later = row_of_key(*arguments(), key_of_lane(block_at(i + (FOUND + (lane >> 1)) * GROUPS)));
#endif
        j = 0;
      }
      s1 = load(block_at(i + GROUPS), found, j + 1);
      use(s0, i);
      i += GROUPS;
      if (i >= end) break;
      s0 = load(block_at(i + GROUPS), found, j + 2);
      use(s1, i);
      i += GROUPS;
      if (i >= end) break;
      j += 2;
    }
  }
  walk.end();
  if constexpr (GROUPS > 1) {
    // the groups' sums meet in the first one, some of the outputs at a time
    constexpr int TURN = 2 * KS <= 8 || BANDS == 1 ? 2 * KS : KS;
    __shared__ float row_m[GROUPS][BANDS][RT][16], row_l[GROUPS][BANDS][RT][16], row_c[GROUPS][BANDS][RT][16];
    __shared__ f32x4_t meet[GROUPS - 1][BANDS][TURN][64];
    if (quad == 0)
#pragma unroll
      for (int t = 0; t < RT; ++t)
        row_m[group][band][t][lane] = walk.ref[t], row_l[group][band][t][lane] = walk.l[t], row_c[group][band][t][lane] = walk.c[t];
    __syncthreads();
    const int r = lane & 15;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float m = -INFINITY, l = 0.f, c = 0.f;
#pragma unroll
      for (int w = 0; w < GROUPS; ++w) m = fmaxf(m, row_m[w][band][t][r]);
#pragma unroll
      for (int w = 0; w < GROUPS; ++w) {
        const float own = row_m[w][band][t][r], by = own == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own - m);
        // a group without a block has no sums; one whose scores are all NaN has sums that are
        l += own == -INFINITY ? row_l[w][band][t][r] : row_l[w][band][t][r] * by;
        c += own == -INFINITY ? row_c[w][band][t][r] : row_c[w][band][t][r] * by;
        if (w == group && own != -INFINITY)
#pragma unroll
          for (int d = 0; d < 2 * KS; ++d) walk.acc[t][d] *= by;
      }
#pragma unroll
      for (int d0 = 0; d0 < 2 * KS; d0 += TURN) {
        if (t + d0 > 0) __syncthreads();  // what met before is read
        if (group > 0)
#pragma unroll
          for (int d = 0; d < TURN; ++d) meet[group - 1][band][d][lane] = walk.acc[t][d0 + d];
        __syncthreads();
        if (group == 0)
#pragma unroll
          for (int d = 0; d < TURN; ++d) {
            f32x4_t others = meet[GROUPS - 2][band][d][lane];
#pragma unroll
            for (int w = GROUPS - 3; w >= 0; --w) others = meet[w][band][d][lane] + others;
            walk.acc[t][d0 + d] += others;
          }
      }
      walk.ref[t] = m, walk.l[t] = l, walk.c[t] = c;
    }
    if (group > 0) return;
  }
#ifdef __HIP_DEVICE_COMPILE__
  const Arguments e = arguments();
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = base + 16 * t + (lane & 15);
    if (r >= rows) continue;
    int token, in_group;
    page_of(PageMagic{e->group.size, e->group.by}, r, token, in_group);
    const size_t row = (size_t)(q0 + token) * e->nq + head * (int)e->group.size + in_group;
    if (e->pieces > 1) {
      float* to = e->part_o + (row * e->pieces + piece) * D;
#pragma unroll
      for (int d = 0; d < 2 * KS; ++d) *(f32x4_t*)(to + 16 * d + 4 * quad) = walk.acc[t][d] + walk.c[t];
      if (quad == 0) *(f32x2_t*)(e->part_ml + 2 * (row * e->pieces + piece)) = (f32x2_t){walk.ref[t], walk.l[t]};
    } else {
      const float by = inverse_sum(walk.ref[t], walk.l[t], e->sink);
      T* to = (T*)e->out + row * D;
#pragma unroll
      for (int d = 0; d < 2 * KS; ++d) store_out4<T>(to + 16 * d + 4 * quad, (walk.acc[t][d] + walk.c[t]) * by);
    }
  }
#endif
}

// The pieces of a row, a block a row: weights of all pieces first, then their sums, every group of D / 4 threads a share of the pieces
// with its loads on their way together. A piece that says it has seen nothing was not written and is not read (its load goes to the first one).
constexpr int MOST_PIECES = 1024;
template <typename T>
__global__ __launch_bounds__(256) void attention4_merge_kernel(T* out, const float* part_o, const float* part_ml, const int* merge_tokens, int nq, int pieces, int sink) {
  constexpr int E = D / 4, GROUPS = 256 / E;
  __shared__ float weight[MOST_PIECES];
  __shared__ f32x4_t sums[GROUPS][E];
  const int lane = threadIdx.x & 63;
  const int index = blockIdx.x / nq, head = blockIdx.x - index * nq;
  const size_t row = (size_t)(merge_tokens ? merge_tokens[index] : index) * nq + head;
  const f32x2_t* ml = (const f32x2_t*)part_ml + row * pieces;
  float m = -INFINITY;  // every wave for itself
  for (int i = lane; i < pieces; i += 64) m = fmaxf(m, ml[i][0]);
  m = wave_max(m);
  float l = 0.f;
  for (int first = 0; first < pieces; first += 64) {
    const int i = first + lane;
    float part = 0.f;
    if (i < pieces) {
      const f32x2_t x = ml[i];
      const float by = x[0] == -INFINITY ? (x[1] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(x[0] - m);  // 1: sums that are NaN
      part = x[1] * by;
      if (threadIdx.x < 64) weight[i] = by;
    }
    l += wave_sum(part);
  }
  __syncthreads();
  const int group = threadIdx.x / E, e = threadIdx.x - group * E;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  if (group < GROUPS) {
    const float* src = part_o + row * pieces * D + 4 * e;
#pragma unroll 8
    for (int i = group; i < pieces; i += GROUPS) {
      const float w = weight[i];
      const f32x4_t x = *(const f32x4_t*)(src + (w == 0.f ? 0 : (size_t)i * D));
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = w == 0.f ? o[k] : fmaf(w, x[k], o[k]);
    }
    sums[group][e] = o;
  }
  __syncthreads();
  if (threadIdx.x >= E) return;
  o = sums[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) o += sums[i][threadIdx.x];
  store_out4<T>(out + row * D + 4 * threadIdx.x, o * inverse_sum(m, l, sink));
}

template <int RT, int NS, int GROUPS, int BANDS, typename T>
static int launch(const Attention4Args& a, hipStream_t stream) {
  const dim3 grid(a.nkv, a.num_tiles, a.pieces);
  const bool by16 = a.page_size % 16 == 0 && (int64_t)a.num_pages * a.nkv * a.page_size * (D / 2 > 8 ? D / 2 : 8) < (1ll << 32);
#define GO(CAP, BY16) attention4_kernel<RT, NS, GROUPS, BANDS, CAP, BY16, T><<<grid, 64 * GROUPS * BANDS, 0, stream>>>(a)
  if (a.softcap > 0.f) {
    if (by16) GO(true, true);
    else GO(true, false);
  } else {
    if (by16) GO(false, true);
    else GO(false, false);
  }
#undef GO
  QRT_LAUNCH_CHECK("attention4");
  if (a.pieces > 1) {
    attention4_merge_kernel<T><<<(unsigned)(a.num_merge_tokens * a.nq), 256, 0, stream>>>((T*)a.out, a.part_o, a.part_ml, a.merge_tokens, a.nq, a.pieces, a.sink);
    QRT_LAUNCH_CHECK("attention4 (merge)");
  }
  return 0;
}

// A tile is 64 / groups * row_tiles rows of a sequence. parts: room for the pieces' sums, behind whose ml_at bytes come their maxima and weights (not
// needed for one piece).
extern "C" int qrt_attention4(const Attention4Plan* plan, const void* q, void* out, const void* k, const void* v, const void* steps, const int* cu_q,
                              const int* kv_lens, const int* table, void* parts, int64_t ml_at, int table_width, int num_pages, int page_size, int sink,
                              float scale, float softcap, int dtype, int groups, int row_tiles, hipStream_t stream) {
  Attention4Args a{*plan, q, out, (const uint8_t*)k, (const uint8_t*)v, (const unsigned*)steps, cu_q, kv_lens, table, (float*)parts,
                         (float*)((char*)parts + ml_at), table_width, num_pages, page_size, sink, scale, softcap, {}, {}};
  QRT_CHECK(dtype == QRT_BF16 || dtype == QRT_F32, "attention4: unknown dtype %d", dtype);
  QRT_CHECK(a.nq > 0 && a.nkv > 0 && a.nq % a.nkv == 0, "attention4: %d query heads on %d key heads", a.nq, a.nkv);
  QRT_CHECK(a.page_size >= 4 && a.page_size % 4 == 0 && a.num_pages > 0 && a.table_width > 0, "attention4: pages of a multiple of 4 tokens, not %d", a.page_size);
  a.page = page_magic(a.page_size), a.group = page_magic(a.nq / a.nkv);
  QRT_CHECK((int64_t)a.num_pages * a.nkv * a.page_size < (1ll << 31), "attention4: a pool of %d pages of %d tokens and %d heads has too many rows", a.num_pages, a.page_size, a.nkv);
  QRT_CHECK(a.window >= 0 && a.chunk >= 0 && a.keep_first >= 0 && !(a.window && a.chunk) && !(a.keep_first && !a.window), "attention4: bad mask");
  QRT_CHECK(a.piece > 0 && a.pieces > 0 && a.pieces <= MOST_PIECES, "attention4: bad pieces %d of %d", a.pieces, a.piece);
  QRT_CHECK(a.pieces == 1 || (a.part_o && ml_at > 0 && ml_at % 16 == 0 && a.num_merge_tokens > 0 && (int64_t)a.num_merge_tokens * a.nq < (1ll << 31)), "attention4: pieces need room for their parts");
  QRT_CHECK(a.tile_seq || !a.tile_row0, "attention4: a list of tiles has sequences and rows");
  QRT_CHECK(a.num_tiles <= 65535, "attention4: %d tiles in one launch, 65535 at most", a.num_tiles);
  QRT_CHECK(((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.steps) % 16 == 0, "attention4: tensors must begin at multiples of 16 bytes");
  if (a.num_tiles <= 0) return 0;
#define ROWS(RT, NS, T)                                        \
  do {                                                         \
    if (groups == 4) return launch<RT, NS, 4, 1, T>(a, stream); \
    if (groups == 2) return launch<RT, NS, 2, 2, T>(a, stream); \
    if (groups == 1) return launch<RT, NS, 1, 4, T>(a, stream); \
  } while (0)
  if (dtype == QRT_F32) {
    if (row_tiles == 1) ROWS(1, 3, float);
  } else if constexpr (D <= 128) {
    if (row_tiles == 2) ROWS(2, 1, bf16_t);
    if (row_tiles == 1 && groups == 4) return launch<1, 1, 4, 1, bf16_t>(a, stream);
  } else {
    if (row_tiles == 1) ROWS(1, 1, bf16_t);
  }
#undef ROWS
  return qrt_fail("attention4: no kernel with %d groups and %d row tiles a wave", groups, row_tiles);
}
