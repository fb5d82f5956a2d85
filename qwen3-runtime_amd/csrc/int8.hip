// Rows to 8-bit integers, and the product of up to 64 such rows with a weight of 8-bit integers.
//
// quantize_rows: a row a block (up to 1,024 columns a wave), held in registers between its maximum and its codes, so memory is
// read once: 2 K bytes in, K out.
//
// int8_rows: few rows stream the weight, which is what bounds them. The MFMA of 16 x 16 x 64 takes 16 bytes of a row a lane, and
// direct loads bring 8 rows x 128 bytes, whole lines, as for bfloat16: the bytes lie alike, two k-steps are 128 columns. A
// block owns 8, 16 or 32 weight rows and all of K, its waves take the steps of 128 columns round-robin, each with a ring of its
// own, and their whole sums meet in LDS; the order of whole sums does not matter. Eight weight rows a block (the operand's other eight
// repeat them) leave the busiest compute unit less to fetch where there are few.
#include "common.h"
#include "direct.h"
#include "gemm_epilogue.h"
#include "int8.h"

// ---------------------------------------------------------------- rows to codes

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_row8(const T* __restrict__ row, int at, int K, float (&v)[8]) {
  if (ALIGNED) {
    if (at < K) {  // K is a multiple of 8 then
      if constexpr (sizeof(T) == 2) {
        const bf16x8_t x = *(const bf16x8_t*)(row + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
      } else {
        const f32x4_t x = *(const f32x4_t*)(row + at), y = *(const f32x4_t*)(row + at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e], v[4 + e] = y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < K ? to_f32<T>(row[at + e]) : 0.f;
  }
}

// THREADS to a row; KEEP pieces of 8 columns a thread stay in registers, wider rows are read a second time.
template <typename T, int THREADS, int KEEP, bool ALIGNED>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scale, int M, int K, int width) {
  __shared__ unsigned part[4];
  const int t = threadIdx.x % THREADS;
  const int row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  const T* src = x + (size_t)min(row, M - 1) * K;
  float v[KEEP][8];
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) load_row8<T, ALIGNED>(src, 8 * (t + THREADS * i), K, v[i]);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(v[i][e]));
  for (int at = 8 * (t + THREADS * KEEP); at < K; at += 8 * THREADS) {
    float w[8];
    load_row8<T, ALIGNED>(src, at, K, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(w[e]));
  }
  most = wave_max_bits(most);
  if (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    most = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  if (row >= M) return;
  const float by = code_factor(most);
  int8_t* out = codes + (size_t)row * width;
  auto store = [&](int at, const float (&w)[8]) {
    typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
    *(u32x2_t*)(out + at) = (u32x2_t){codes4(w[0], w[1], w[2], w[3], by), codes4(w[4], w[5], w[6], w[7], by)};
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = 8 * (t + THREADS * i);
    if (at < width) store(at, v[i]);
  }
  for (int at = 8 * (t + THREADS * KEEP); at < width; at += 8 * THREADS) {
    float w[8];
    load_row8<T, ALIGNED>(src, at, K, w);
    store(at, w);
  }
  if (t == 0) scale[row] = row_scale_of(most);
}

template <typename T>
static void launch_quantize(const T* x, int8_t* codes, float* scale, int M, int K, int width, hipStream_t stream) {
  const bool aligned = K % 8 == 0 && (uintptr_t)x % 16 == 0;
#define GO(THREADS, KEEP, ALIGNED) \
  quantize_rows_kernel<T, THREADS, KEEP, ALIGNED><<<dim3((M + 256 / THREADS - 1) / (256 / THREADS)), dim3(256), 0, stream>>>(x, codes, scale, M, K, width)
  if (!aligned) GO(256, 4, false);
  else if (width <= 1024) GO(64, 2, true);
  else if (width <= 4096) GO(256, 2, true);
  else GO(256, 5, true);
#undef GO
}

static int check_width(const char* name, int M, int K, int width) {
  QRT_CHECK(M >= 0 && K > 0 && width >= K && width % INT8_STAGE == 0 && width <= INT8_MOST_WIDTH, "%s: bad sizes M=%d K=%d, rows of %d", name, M, K, width);
  return 0;
}

// codes [M, width] (columns K and on are zeros), scale [M]; width: K up to a multiple of 128
extern "C" int qrt_quantize_rows(const void* x, int dtype, void* codes, float* scale, int M, int K, int width, hipStream_t stream) {
  if (check_width("quantize_rows", M, K, width)) return -1;
  QRT_CHECK(dtype == QRT_BF16 || dtype == QRT_F32, "quantize_rows: unknown dtype %d", dtype);
  QRT_CHECK((uintptr_t)codes % 16 == 0, "quantize_rows: codes must begin at a multiple of 16 bytes");
  if (M == 0) return 0;
  if (dtype == QRT_BF16) launch_quantize((const bf16_t*)x, (int8_t*)codes, scale, M, K, width, stream);
  else launch_quantize((const float*)x, (int8_t*)codes, scale, M, K, width, stream);
  QRT_LAUNCH_CHECK("quantize_rows");
  return 0;
}

// ---------------------------------------------------------------- few rows

struct Int8Rows {
  const void* x;        // FUSED: rows as they are [M, K]
  const int8_t* a;      // otherwise their codes [M, width] and scales [M]
  const float* a_scale;
  const int8_t* w;      // [N or 2 N, width]
  const float* w_scale;
  void* c;
  int M, N, K, width;
  GatedEpilogue ep;
};

// The waves' share of the rows that a FUSED block turns into codes: pieces of 8 columns a lane, in registers from the loads to the codes.
constexpr int FUSED_PIECES = 10;
// Waves that share a row's maximum.
constexpr int fused_parts(int M) { return M == 1 ? 4 : M == 2 ? 2 : 1; }
constexpr int fused_steps(int M, int width) { return (width / 8 + 64 * fused_parts(M) - 1) / (64 * fused_parts(M)); }
constexpr bool fused_takes(int M, int width) { return M <= 16 && (M * fused_parts(M) + 3) / 4 * fused_steps(M, width) <= FUSED_PIECES; }

// NW waves; WU units of eight weight rows (1: the operand's rows 8 to 15 repeat the others); MB blocks of 16 rows of the
// activations (FEW: eight); GATED: half of the units are gate rows, half the up rows that belong to them.
template <int NW, int WU, int MB, bool FEW, int U, bool GATED, bool FUSED, typename TX, typename TO>
__global__ __launch_bounds__(64 * NW) void int8_rows_kernel(Int8Rows p) {
  constexpr int NT = WU == 1 ? 1 : WU / 2, AU = FEW ? 1 : 2 * MB, LOADS = WU + (FUSED ? 0 : AU), SLOT = LOADS * 1024;
  constexpr int OUTS = GATED ? 4 * WU : 8 * WU, ONCE = 2;  // outputs of a block; the cache policy of a non-temporal load
  static_assert((U - 1) * LOADS < 64, "the loads' counter holds 63");
  static_assert(!FUSED || (NW == 4 && MB == 1), "the waves that share a row are counted for four");
  extern __shared__ __align__(16) unsigned char rows_lds[];  // [NW][U] slots, later the sums; FUSED: the rows' codes behind them
  __shared__ unsigned most_of[FUSED ? 16 : 1];
  const int lane = threadIdx.x & 63, wave = uniform_wave_number();
  const int r16 = lane & 15, quad = lane >> 4, sub = lane >> 3, piece = (lane & 7) ^ sub;
  const int n0 = blockIdx.x * OUTS;
  unsigned char* ring = rows_lds + (size_t)wave * U * SLOT;
  constexpr size_t MEET = (size_t)NW * NT * MB * 1024, RINGS = (size_t)NW * U * SLOT;
  unsigned char* const own_codes = rows_lds + (RINGS > MEET ? RINGS : MEET);
  const int width = p.width, steps = width / INT8_STAGE;

  // FUSED: the rows come first, and are waited for behind the weights' loads
  float v[FUSED ? FUSED_PIECES : 1][8];
  const int parts = fused_parts(p.M), its = fused_steps(p.M, width), items = p.M * parts;
  auto item_of = [&](int j, int& row, int& at) {  // piece j of this lane: its row (p.M or more: none) and first column
    const int item = wave + NW * (j / its);
    row = item / parts;
    at = 8 * ((item % parts) * 64 + lane + 64 * parts * (j % its));
    return item < items;
  };
  if constexpr (FUSED) {
#pragma unroll
    for (int j = 0; j < FUSED_PIECES; ++j) {
      int row, at;
      const bool any = item_of(j, row, at);
      load_row8<TX, true>((const TX*)p.x + (size_t)(any ? row : 0) * p.K, any ? at : p.K, p.K, v[j]);
    }
  }
  const int8_t* src[LOADS];
#pragma unroll
  for (int u = 0; u < WU; ++u) {  // rows past the end repeat the last; not stored
    const int up = GATED && (WU == 2 ? u == 1 : u >= WU / 2);
    const int unit = GATED ? (WU == 2 ? 0 : u % (WU / 2)) : u;
    src[u] = p.w + (size_t)(min(n0 + 8 * unit + sub, p.N - 1) + (up ? p.N : 0)) * width + 16 * piece;
  }
  if constexpr (!FUSED) {
#pragma unroll
    for (int u = 0; u < AU; ++u) src[WU + u] = p.a + (size_t)min(8 * u + sub, p.M - 1) * width + 16 * piece;
  }
  const int mine = max(0, (steps - wave + NW - 1) / NW);
  auto fetch = [&](int i, int slot) {
    const size_t at = (size_t)(wave + i * NW) * INT8_STAGE;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      if (u < WU) __builtin_amdgcn_global_load_lds((global_ptr_t)(src[u] + at), (lds_ptr_t)(ring + slot * SLOT + u * 1024), 16, 0, ONCE);
      else __builtin_amdgcn_global_load_lds((global_ptr_t)(src[u] + at), (lds_ptr_t)(ring + slot * SLOT + u * 1024), 16, 0, 0);
    }
  };
  int fetched = 0;
  for (; fetched < U && fetched < mine; ++fetched) fetch(fetched, fetched);

  if constexpr (FUSED) {
    __shared__ unsigned part_of[64];
    unsigned most = 0;
#pragma unroll
    for (int j = 0; j < FUSED_PIECES; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(v[j][e]));
      if (j % its == its - 1) {  // the same in every lane
        const unsigned m = wave_max_bits(most);
        const int item = wave + NW * (j / its);
        if (lane == 0 && item < items) part_of[item] = m;
        most = 0;
      }
    }
    QRT_WAIT_LDS();
    QRT_BARRIER();
#pragma unroll
    for (int j = 0; j < FUSED_PIECES; ++j) {
      int row, at;
      if (!item_of(j, row, at) || at >= width) continue;
      unsigned m = 0;
      for (int i = 0; i < parts; ++i) m = max(m, part_of[row * parts + i]);
      if (at == 0) most_of[row] = m;
      const float by = code_factor(m);
      typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
      // piece c of 16 columns of a stage's row r lies at 16 (c ^ (r & 7)), as in the rings
      unsigned char* to = own_codes + (size_t)(at >> 7) * (FEW ? 1024 : 2048) + row * 128 + 16 * (((at >> 4) & 7) ^ (row & 7)) + (at & 8);
      *(u32x2_t*)to = (u32x2_t){codes4(v[j][0], v[j][1], v[j][2], v[j][3], by), codes4(v[j][4], v[j][5], v[j][6], v[j][7], by)};
    }
    QRT_WAIT_LDS();
    QRT_BARRIER();
  }

  i32x4_t acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[t][b] = (i32x4_t){0, 0, 0, 0};
  const int rw = WU == 1 ? r16 & 7 : r16, ra = FEW ? r16 & 7 : r16;
  const int w_at[2] = {rw * 128 + 16 * (quad ^ (r16 & 7)), rw * 128 + 16 * ((4 + quad) ^ (r16 & 7))};
  const int a_at[2] = {ra * 128 + 16 * (quad ^ (r16 & 7)), ra * 128 + 16 * ((4 + quad) ^ (r16 & 7))};
  int slot = 0;
  for (int i = 0; i < mine; ++i) {
    // step i has landed when at most the U - 1 steps fetched after it are still on their way
    if (fetched - i == U) QRT_WAIT_LOADS((U - 1) * LOADS);
    else QRT_WAIT_LOADS(0);
    const unsigned char* at = ring + slot * SLOT;
    const unsigned char* codes = FUSED ? own_codes + (size_t)(wave + i * NW) * (FEW ? 1024 : 2048) : at + WU * 1024;
    i32x4_t w[NT][2], a[MB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < NT; ++t) w[t][h] = *(const i32x4_t*)(at + t * 2048 + w_at[h]);
#pragma unroll
      for (int b = 0; b < MB; ++b) a[b][h] = *(const i32x4_t*)(codes + b * 2048 + a_at[h]);
    }
    QRT_WAIT_LDS();  // the slot is in registers: the next step may overwrite it
    if (fetched < mine) {
      fetch(fetched, slot);
      ++fetched;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = IntProducts::add(w[t][h], a[b][h], acc[t][b]);
    slot = slot + 1 == U ? 0 : slot + 1;
  }
  __syncthreads();  // every wave has read its last slot: the rings' room now takes the sums
  int* red = (int*)rows_lds;  // [NW][NT][MB][4][64]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[(((wave * NT + t) * MB + b) * 4 + r) * 64 + lane] = acc[t][b][r];
  __syncthreads();
  // sum r of (tile, block, lane l): weight row 16 t + 4 (l / 16) + r, row 16 b + (l & 15)
  auto total = [&](int t, int b, int l, int r) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += red[(((w * NT + t) * MB + b) * 4 + r) * 64 + l];
    return (float)s;
  };
  constexpr int TILES_OUT = GATED && NT > 1 ? NT / 2 : NT;
  for (int i = threadIdx.x; i < TILES_OUT * MB * 256; i += 64 * NW) {
    const int l = i & 63, r = (i >> 6) & 3, b = (i >> 8) % MB, t = (i >> 8) / MB;
    const int m = 16 * b + (l & 15), in_tile = 4 * (l >> 4) + r;
    if (m >= p.M || (OUTS < 16 && in_tile >= OUTS)) continue;
    const int n = n0 + 16 * t + in_tile;
    if (n >= p.N) continue;
    const float sx = FUSED ? row_scale_of(most_of[m]) : p.a_scale[m];
    float y = total(t, b, l, r) * sx * p.w_scale[n];
    if constexpr (GATED) {
      const float u = total(NT > 1 ? t + NT / 2 : t, b, NT > 1 ? l : l + 32, r) * sx * p.w_scale[p.N + n];
      y = gated_act(y, u, p.ep.kind, p.ep.limit);
    }
    ((TO*)p.c)[(size_t)m * p.N + n] = from_f32<TO>(y);
  }
}

template <int NW, int WU, int MB, bool FEW, int U, bool GATED, bool FUSED, typename TX, typename TO>
static int launch_int8_rows(const Int8Rows& p, hipStream_t stream) {
  constexpr int NT = WU == 1 ? 1 : WU / 2, AU = FEW ? 1 : 2 * MB, OUTS = GATED ? 4 * WU : 8 * WU;
  constexpr size_t rings = (size_t)NW * U * (WU + (FUSED ? 0 : AU)) * 1024, meet = (size_t)NW * NT * MB * 1024;
  const size_t smem = (rings > meet ? rings : meet) + (FUSED ? (size_t)p.width / INT8_STAGE * AU * 1024 : 0);
  static_assert(rings <= 156 * 1024, "the rings of this configuration do not fit LDS");
  QRT_CHECK(smem <= 156 * 1024, "int8_rows: %d columns need %zu bytes of LDS", p.width, smem);
  auto kernel = int8_rows_kernel<NW, WU, MB, FEW, U, GATED, FUSED, TX, TO>;
  static bool allowed = false;  // once per kernel: not inside a stream capture again and again
  if (!allowed) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 156 * 1024) != hipSuccess)
      return qrt_fail("int8_rows: cannot get LDS");
    allowed = true;
  }
  kernel<<<dim3((p.N + OUTS - 1) / OUTS), dim3(64 * NW), smem, stream>>>(p);
  QRT_LAUNCH_CHECK("int8_rows");
  return 0;
}

template <bool GATED, bool FUSED, typename TX, typename TO>
static int rows_by_size(const Int8Rows& p, hipStream_t stream) {
  if constexpr (FUSED) {
    if (p.M <= 8) return launch_int8_rows<4, GATED ? 2 : 1, 1, true, 4, GATED, true, TX, TO>(p, stream);
    return launch_int8_rows<4, 2, 1, false, 4, GATED, true, TX, TO>(p, stream);
  } else {
    if (p.M <= 8) return launch_int8_rows<4, 2, 1, true, 4, GATED, false, TX, TO>(p, stream);
    if (p.M <= 16) return launch_int8_rows<4, 2, 1, false, 4, GATED, false, TX, TO>(p, stream);
    if (p.M <= 32) return launch_int8_rows<4, 2, 2, false, 4, GATED, false, TX, TO>(p, stream);
    if (p.M <= 48) return launch_int8_rows<4, 4, 3, false, 3, GATED, false, TX, TO>(p, stream);
    return launch_int8_rows<4, 4, 4, false, 3, GATED, false, TX, TO>(p, stream);
  }
}

// Whether qrt_int8_rows turns these rows into codes itself.
extern "C" int qrt_int8_rows_fuses(int M, int K, int width) { return M > 0 && K % 8 == 0 && fused_takes(M, width); }

// c [M, N] of up to 64 rows. Either x (rows as they are, in x_dtype; qrt_int8_rows_fuses says which) or a and a_scale. act_kind < 0: no gate;
// otherwise w is [2 N, width].
extern "C" int qrt_int8_rows(const void* x, int x_dtype, const void* a, const float* a_scale, const void* w, const float* w_scale, void* c,
                             int out_dtype, int M, int N, int K, int width, int act_kind, float limit, hipStream_t stream) {
  if (check_width("int8_rows", M, K, width)) return -1;
  QRT_CHECK(N > 0 && M <= 64, "int8_rows: bad sizes M=%d N=%d", M, N);
  QRT_CHECK(act_kind <= QRT_ACT_CLAMPED, "int8_rows: unknown activation %d", act_kind);
  QRT_CHECK(out_dtype == QRT_BF16 || out_dtype == QRT_F32, "int8_rows: unknown output dtype %d", out_dtype);
  QRT_CHECK(((uintptr_t)(x ? x : a) | (uintptr_t)w) % 16 == 0, "int8_rows: operands must begin at multiples of 16 bytes");
  QRT_CHECK(!x || qrt_int8_rows_fuses(M, K, width), "int8_rows: %d rows of %d columns come as codes", M, K);
  QRT_CHECK(!x || x_dtype == QRT_BF16 || x_dtype == QRT_F32, "int8_rows: unknown dtype %d", x_dtype);
  if (M == 0) return 0;
  const Int8Rows p{x, (const int8_t*)a, a_scale, (const int8_t*)w, w_scale, c, M, N, K, width, GatedEpilogue{act_kind, limit, nullptr}};
  const bool bf = out_dtype == QRT_BF16;
#define GO(GATED)                                                                                                            \
  do {                                                                                                                       \
    if (x && x_dtype == QRT_BF16) return bf ? rows_by_size<GATED, true, bf16_t, bf16_t>(p, stream) : rows_by_size<GATED, true, bf16_t, float>(p, stream); \
    if (x) return bf ? rows_by_size<GATED, true, float, bf16_t>(p, stream) : rows_by_size<GATED, true, float, float>(p, stream);                         \
    return bf ? rows_by_size<GATED, false, float, bf16_t>(p, stream) : rows_by_size<GATED, false, float, float>(p, stream);  \
  } while (0)
  if (act_kind >= 0) GO(true);
  GO(false);
#undef GO
}
