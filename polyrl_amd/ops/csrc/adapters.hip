// Low-rank adapters of many requests beside one shared projection:
//
//   out[t, n] = y[t, n] + s_i sum_j b[i, n, j] (sum_k a[i, p(n), j, k] x[t, k])
//
// with i the adapter of row t's request and p(n) the part of a fused projection (q, k, v)
// that column n belongs to.  Rows without an adapter are y's.
//
// Three steps.  ``adapter_plan`` (once a step of a model, for all its projections) puts
// the rows in the order of their adapters and cuts them into tiles of rows that share
// one; all on the device, so that a captured decode step finds its tiles again.  ``down``
// forms h = A x, the inner dimension cut over a block's waves and, where there are few
// tiles, over blocks; ``up`` adds the blocks' shares in their order, multiplies with B
// and adds the result to y, which it reads and writes once.  (One kernel for both would
// read A in every block of columns; h is 1% of y.)
//
// What bounds it: memory, prompts by y and out (6504 rows, ranks 32, the four projections of
// 4096 / 6144 / 14336 numbers, 1.43 GB: 373 us, 3.8 TB/s; the widest, 746 MB, 152 to 157 us,
// where a copy of the same tiles takes 131), decode by the adapters (57 rows of as many adapters
// of ranks 64 and 32, 0.45 GB: 149 us, 3.0 TB/s; a wave of ``down`` has one round of its loads on
// its way); one row by nine launches, 34 us in a graph and 35 to 45 issued one by one.
//
// Matrix cores: 16x16x32 in bf16, 16x16x4 in fp32.  h is a sum in 32 bits; as an operand
// in bf16 it is cut into three bf16 numbers of 8 bits each, whose sum is h, each with its own
// product, so that nothing is lost of it (two would lose 2^-16, one 2^-8).
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"
#include "rows_overlap.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

// A lane's 16 bytes of an operand: numbers k .. k + PER of row (or column) l % 16, with
// k = PER * (l / 16) inside a step of 4 * PER
template <typename T> struct Operand;
template <> struct Operand<__bf16> {
  static constexpr int PER = 8, STEP = 32;
  DEV_INLINE static f32x4_t mul(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
};
template <> struct Operand<float> {
  static constexpr int PER = 4, STEP = 16;
  // (the order of the inner dimension is the same one in both operands)
  DEV_INLINE static f32x4_t mul(const i32x4_t& a, const i32x4_t& b, f32x4_t c) {
    const f32x4_t u = __builtin_bit_cast(f32x4_t, a), v = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[j], v[j], c, 0, 0, 0);
    return c;
  }
};

// p[0 .. have) of a lane's numbers, zeros behind.  WORDS: 16 bytes at p can be read
// wherever have > 0
template <typename T, bool WORDS>
DEV_INLINE i32x4_t load_some(const T* p, int have) {
  constexpr int PER = Operand<T>::PER;
  if (have <= 0) return i32x4_t{0, 0, 0, 0};
  T v[PER];
  if (WORDS) {
    const i32x4_t w = *reinterpret_cast<const i32x4_t*>(p);
    if (have >= PER) return w;
    __builtin_memcpy(v, &w, 16);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j < have) v[j] = p[j];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (j >= have) v[j] = (T)0.f;
  i32x4_t w;
  __builtin_memcpy(&w, v, 16);
  return w;
}

// ---------------------------------------------------------------------- plan
// plan: the number of tiles; for each one (4 ints) its adapter, its number of rows and that
// of the rows of the tiles before it, where its part of h is; for each one its rows, in
// places for a whole tile, so that a block knows where to read them before it knows anything
// else.  Rows without an adapter come last, as tiles of adapter -1.
constexpr int PLAN_HEAD = 4;
constexpr int MOST_SLOTS = 4095, MOST_RANK = 256;

// the sum of the wave's lower lanes' numbers and this one's
DEV_INLINE int wave_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int below = __shfl_up(x, d, 64);
    if (lane >= d) x += below;
  }
  return x;
}

// f(row, adapter, lanes): every row, with the lanes of the wave whose rows are of the same
// adapter, as far as two rounds find them (a prompt's rows are all of one), else its own
template <typename F>
DEV_INLINE void by_adapter(const int* index, int T, int slots, F f) {
  constexpr int U = 8;
  for (int t0 = 0; t0 < T; t0 += U * 1024) {
    int s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * 1024 + threadIdx.x;
      s[u] = t < T ? index[t] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * 1024 + threadIdx.x;
      if (t0 + u * 1024 >= T) break;
      if (s[u] < 0 || s[u] >= slots) s[u] = slots;
      bool mine = t < T;
      for (int r = 0; r < 2; ++r) {
        const unsigned long long left = __ballot(mine);
        if (left == 0) break;
        const int first = __shfl(s[u], __ffsll(left) - 1, 64);
        const bool now = mine && s[u] == first;
        const unsigned long long same = __ballot(now);
        if (now) f(t, s[u], same);
        mine = mine && !now;
      }
      if (mine) f(t, s[u], 1ull << (threadIdx.x & 63));
    }
  }
}

__global__ __launch_bounds__(1024) void adapter_plan_kernel(int* plan, const int* index,
                                                            int T, int slots, int tile,
                                                            int most) {
  __shared__ int count[MOST_SLOTS + 1], cursor[MOST_SLOTS + 1];
  __shared__ int sums[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  for (int s = tid; s <= slots; s += 1024) count[s] = 0;
  __syncthreads();
  by_adapter(index, T, slots, [&](int, int s, unsigned long long lanes) {
    if (__ffsll(lanes) - 1 == lane) atomicAdd(&count[s], __popcll(lanes));
  });
  __syncthreads();
  // each thread a stretch of adapters, then the tiles of the threads before
  const int per = (slots + 1 + 1023) / 1024;
  int tiles = 0, rows = 0;
  for (int s = tid * per; s < min((tid + 1) * per, slots + 1); ++s) {
    tiles += (count[s] + tile - 1) / tile;
    rows += count[s];
  }
  int n = wave_scan(tiles), before = wave_scan(rows);
  if (lane == 63) sums[0][wid] = n, sums[1][wid] = before;
  __syncthreads();
  for (int w = 0; w < wid; ++w) n += sums[0][w], before += sums[1][w];
  if (tid == 1023) plan[0] = n;
  n -= tiles, before -= rows;
  i32x4_t* entry = reinterpret_cast<i32x4_t*>(plan + PLAN_HEAD);
  for (int s = tid * per; s < min((tid + 1) * per, slots + 1); ++s) {
    cursor[s] = n * tile;
    for (int i = 0; i < count[s]; i += tile, ++n)
      entry[n] = i32x4_t{s < slots ? s : -1, min(tile, count[s] - i), before + i, 0};
    before += count[s];
  }
  __syncthreads();
  int* order = plan + PLAN_HEAD + 4 * most;
  by_adapter(index, T, slots, [&](int t, int s, unsigned long long lanes) {
    const int first = __ffsll(lanes) - 1;
    int place = 0;
    if (first == lane) place = atomicAdd(&cursor[s], __popcll(lanes));
    place = __builtin_amdgcn_ds_bpermute(first * 4, place);
    order[place + __popcll(lanes & ((1ull << lane) - 1))] = t;
  });
}

// ---------------------------------------------------------------------- down
struct Shape {
  int T, K, N, parts, rank, rank16;   // rank16: rank rounded up to whole tiles of 16
  long ldx, ldy, ldo;
  int split, most;                    // shares of the inner dimension; places for tiles
  int first[9];                       // columns of the parts
};

constexpr int MOST_SPLIT = 4;

// Operand tiles from rows that lie far apart.  The matrix cores want row l % 16 in lane l,
// but the L1 takes a cycle for each lane of a load whose neighbours do not lie beside it
// and 16 for four rows of 256 bytes (a kernel of loads alone, 6528 rows of 14336 bf16
// numbers and 32 of A for every 32 of them: 57 us by lanes of 16 rows, 42 by 8 rows of 128
// bytes, 41 by 4 of 256; this kernel 72 and 52).  So load j reads rows 4 * i + j, i = 0 .. 3,
// a lane 16 bytes of row 4 * (l / 4 % 4) + j from 64 * (l / 16) + 16 * (l % 4), and every four
// lanes transpose what they have: then load j's register holds row l % 16, bytes
// 64 * (l / 16) + 16 * j.  (The order of the inner dimension is the same in both operands.)
DEV_INLINE void quads_transposed(i32x4_t (&v)[4]) {
  const bool one = threadIdx.x & 1, two = threadIdx.x & 2;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
#pragma unroll
    for (int p = 0; p < 4; p += 2) {    // lane bit 0 and load bit 0
      const int a = v[p][d], b = v[p + 1][d];
      const int na = __builtin_amdgcn_mov_dpp(a, 0xb1, 0xf, 0xf, true);
      const int nb = __builtin_amdgcn_mov_dpp(b, 0xb1, 0xf, 0xf, true);
      v[p][d] = one ? nb : a;
      v[p + 1][d] = one ? b : na;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {       // and 1
      const int a = v[p][d], b = v[p + 2][d];
      const int na = __builtin_amdgcn_mov_dpp(a, 0x4e, 0xf, 0xf, true);
      const int nb = __builtin_amdgcn_mov_dpp(b, 0x4e, 0xf, 0xf, true);
      v[p][d] = two ? nb : a;
      v[p + 2][d] = two ? b : na;
    }
  }
}

// h[share][row in the tiles' order][part][j].  A block takes RT * 16 rows of a tile, CT tiles of 16 ranks
// (tile i: ranks 16 * (i / parts) .. of part i % parts) and a share of the inner
// dimension, each of its NW waves a part of that
template <typename T, int NW, int RT, int CT, bool WORDS>
__global__ __launch_bounds__(NW * 64) void adapter_down_kernel(
    float* __restrict__ h, const T* __restrict__ x, const T* __restrict__ a,
    const int* __restrict__ ranks, const int* __restrict__ plan, const Shape z,
    int subs) {
  using O = Operand<T>;
  __shared__ float red[NW * RT * CT * 256];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int l15 = lane & 15, lhi = lane >> 4;
  const int groups = (z.rank16 / 16 * z.parts + CT - 1) / CT;
  int id = blockIdx.x;
  const int share = id % z.split;
  id /= z.split;
  const int group = id % groups, at = id / groups, tile = at / subs;
  // Two steps of reads that wait for each other: the tile and its rows; what they name.
  // (Rows past the tile and ranks past the adapter's are any, dropped below.)
  const int place = at * RT * 16;
  const int* order = plan + PLAN_HEAD + 4 * z.most + place;
  const int first = lane / 4 % 4 * 4, part_of = (lhi * 4 + lane % 4) * O::PER;
  int row[RT][4];                     // rows of load j
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) row[r][j] = order[r * 16 + first + j];
  const i32x4_t t = reinterpret_cast<const i32x4_t*>(plan + PLAN_HEAD)[tile];
  const int slot = t[0], rows = t[1] - at % subs * RT * 16;
  if (tile >= plan[0] || slot < 0 || rows <= 0) return;
  const int rank = ranks ? min(max(ranks[slot], 0), z.rank) : z.rank;
  const int some = __builtin_amdgcn_readfirstlane(row[0][0]);
  const T* xr[RT][4];
  const T* base[CT];
  uint32_t ar[CT][4];                 // (a matrix is less than 2^30 bytes)
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      xr[r][j] = x + (long)(r * 16 + first + j < rows ? row[r][j] : some) * z.ldx + part_of;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int i = group * CT + c;
    base[c] = a + ((long)slot * z.parts + i % z.parts) * z.rank * z.K;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      ar[c][j] = (uint32_t)min(i / z.parts * 16 + first + j, z.rank - 1) * (uint32_t)z.K +
                 (uint32_t)part_of;
  }
  if (group * CT / z.parts * 16 >= rank) return;
  f32x4_t acc[RT][CT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[r][c] = {0.f, 0.f, 0.f, 0.f};
  // this wave's part of the inner dimension, 256 bytes a round
  constexpr int ROUND = 4 * O::STEP;
  const int rounds = (z.K + ROUND - 1) / ROUND;
  const int per = (rounds + z.split * NW - 1) / (z.split * NW) * ROUND;
  const int k0 = (share * NW + wid) * per, k1 = min(k0 + per, z.K);
  auto round = [&](int k, auto whole) {
    i32x4_t xv[RT][4], av[CT][4];
    const int have = decltype(whole)::value ? O::PER : k1 - k - part_of;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
        av[c][j] = load_some<T, WORDS>(base[c] + k + ar[c][j], have);
#pragma unroll
      for (int r = 0; r < RT; ++r) xv[r][j] = load_some<T, WORDS>(xr[r][j] + k, have);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) quads_transposed(av[c]);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      quads_transposed(xv[r]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = O::mul(xv[r][j], av[c][j], acc[r][c]);
    }
  };
  int k = k0;
#pragma unroll 1
  for (; k + ROUND <= k1; k += ROUND) round(k, std::true_type());
  if (k < k1) round(k, std::false_type());
  // sums of the waves; register i: row 4 * (lane / 16) + i, column lane % 16
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[((wid * RT + r) * CT + c) * 256 + (lhi * 4 + i) * 16 + l15] = acc[r][c][i];
  __syncthreads();
  for (int o = threadIdx.x; o < RT * CT * 256; o += NW * 64) {
    const int i = group * CT + o / 256 % CT, r = o / 256 / CT;
    const int j = i / z.parts * 16 + o % 16;
    if (r * 16 + o % 256 / 16 >= rows || j >= rank) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w * RT * CT * 256 + o];
    h[(((long)share * z.T + t[2] + at % subs * RT * 16 + r * 16 + o % 256 / 16) * z.parts +
       i % z.parts) * z.rank16 + j] = v;
  }
}

// ------------------------------------------------------------------------ up
// h's numbers j .. j + 4 of a row, times s (the shares' sums in their order, zeros from rank
// on), as PARTS numbers of type T whose sum they are: of bf16 each the upper 8 bits of what
// those before it leave, cut and not rounded, so that none is larger than h
template <typename T> constexpr int PARTS = sizeof(T) == 2 ? 3 : 1;

template <typename T>
struct Four {
  T part[PARTS<T>][4];
  DEV_INLINE Four(f32x4_t v, float s, int left) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f = e < left ? v[e] * s : 0.f;
      if (PARTS<T> == 1) {
        part[0][e] = (T)f;
        continue;
      }
#pragma unroll
      for (int p = 0; p < PARTS<T>; ++p) {
        const float cut = __uint_as_float(__float_as_uint(f) & 0xffff0000u);
        part[p][e] = (T)cut;
        f = isfinite(f) ? f - cut : 0.f;    // (an infinite h has no lower part)
      }
    }
  }
  DEV_INLINE void put(int p, T* at) const {
    struct alignas(sizeof(T) * 4) Word { T v[4]; };
    Word w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.v[e] = part[p][e];
    *reinterpret_cast<Word*>(at) = w;
  }
};
DEV_INLINE f32x4_t shares_sum(const float* p, long share, int split) {
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < MOST_SPLIT; ++w)
    if (w < split) v += *reinterpret_cast<const f32x4_t*>(p + w * share);
  return v;
}

// Where a block of ``wide`` columns stands: a tile, a part and its columns n0 .. end
struct Place {
  int tile, part, n0, end;
  DEV_INLINE Place(const Shape& z, int cols, int wide) : tile(blockIdx.x / cols), part(0) {
    int col = blockIdx.x % cols;
    while (col >= (z.first[part + 1] - z.first[part] + wide - 1) / wide) {
      col -= (z.first[part + 1] - z.first[part] + wide - 1) / wide;
      ++part;
    }
    n0 = z.first[part] + col * wide, end = z.first[part + 1];
  }
};

// Few rows: a tile of 16, where b is most of what is read.  A wave takes 64 columns, b
// straight into its operands, as four tiles whose columns are dealt so that a lane holds
// whole 16-byte words of its row l % 16: word q is columns 4 * VEC * q + VEC * (l / 16) ..
// WORDS: rows of b come in whole 16-byte words; OUT_WORDS: those of y and out
constexpr int FEW_COLS = 256, FEW_RANK = 64;

template <typename T, bool WORDS, bool OUT_WORDS>
__global__ __launch_bounds__(256) void adapter_up_few_kernel(
    T* out, const T* y, const float* __restrict__ h, const T* __restrict__ b,
    const float* __restrict__ scale, const int* __restrict__ ranks,
    const int* __restrict__ plan, const Shape z, int cols) {
  using O = Operand<T>;
  constexpr int VEC = 16 / (int)sizeof(T), Q = 16 / VEC, PER_Q = VEC / 4;
  constexpr int PITCH = FEW_RANK + VEC, S = FEW_RANK / O::STEP;
  struct alignas(16) Word { T v[VEC]; };
  __shared__ __attribute__((aligned(16))) T hs[PARTS<T>][16][PITCH];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int l15 = lane & 15, lhi = lane >> 4;
  const Place at(z, cols, FEW_COLS);
  const int place = at.tile * 16;
  const int own = (plan + PLAN_HEAD + 4 * z.most + place)[l15];
  const i32x4_t t = reinterpret_cast<const i32x4_t*>(plan + PLAN_HEAD)[at.tile];
  const int slot = t[0], rows = t[1];
  if (at.tile >= plan[0] || (slot < 0 && out == y)) return;
  const int rank = slot < 0 ? 0 : ranks ? min(max(ranks[slot], 0), z.rank) : z.rank;
  const int n0 = at.n0 + wid * 64, end = at.end;
  const bool whole = OUT_WORDS && n0 + 64 <= end;
  // all that is read is on its way before any of it is waited for
  // (by all lanes: inside the choice it would be the first lane past the tile's)
  const int some = __builtin_amdgcn_readfirstlane(own);
  const long row = l15 < rows ? own : some;
  const T* bb = b + (long)max(slot, 0) * z.N * z.rank;
  i32x4_t bv[S][4];
  auto load_b = [&](int j0) {
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
      for (int c = 0; c < 4; ++c) {               // columns past the part: its last
        const int n = n0 + c / PER_Q * 4 * VEC + l15 / 4 * VEC + c % PER_Q * 4 + l15 % 4;
        const int j = j0 + k * O::STEP + lhi * O::PER;
        bv[k][c] = load_some<T, WORDS>(bb + (long)min(n, end - 1) * z.rank + j, rank - j);
      }
  };
  load_b(0);
  Word yv[Q];
  if (whole)
#pragma unroll
    for (int q = 0; q < Q; ++q)
      yv[q] = *reinterpret_cast<const Word*>(y + row * z.ldy + n0 + q * 4 * VEC + lhi * VEC);
  const float s = slot < 0 ? 0.f : scale[slot];
  f32x4_t acc[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int j0 = 0; j0 < rank; j0 += FEW_RANK) {
    if (j0 > 0) {
      load_b(j0);
      __syncthreads();
    }
    const int r = threadIdx.x / 16, j = threadIdx.x % 16 * 4;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (r < rows && j0 + j < rank)
      v = shares_sum(h + (((long)t[2] + r) * z.parts + at.part) * z.rank16 + j0 + j,
                     (long)z.T * z.parts * z.rank16, z.split);
    const Four<T> f(v, s, rank - j0 - j);
#pragma unroll
    for (int p = 0; p < PARTS<T>; ++p) f.put(p, &hs[p][r][j]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; ++k) {
      if (j0 + k * O::STEP >= rank) break;
#pragma unroll
      for (int p = 0; p < PARTS<T>; ++p) {
        const i32x4_t hv =
            *reinterpret_cast<const i32x4_t*>(&hs[p][l15][k * O::STEP + lhi * O::PER]);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = O::mul(bv[k][c], hv, acc[c]);
      }
    }
  }
  if (l15 >= rows || (rank == 0 && out == y)) return;
  // register i of tile c: row lane % 16, column 4 * (lane / 16) + i of the tile's
  if (whole) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      Word w = yv[q];
      if (rank > 0)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          w.v[e] = (T)((float)w.v[e] + acc[q * PER_Q + e / 4][e % 4]);
      *reinterpret_cast<Word*>(out + row * z.ldo + n0 + q * 4 * VEC + lhi * VEC) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int n = n0 + i / VEC * 4 * VEC + lhi * VEC + i % VEC;
      if (n >= end) continue;
      const T old = y[row * z.ldy + n];
      out[row * z.ldo + n] = rank > 0 ? (T)((float)old + acc[i / 4][i % 4]) : old;
    }
  }
}

// Many rows, where y and out are most of it: a block takes a tile of 64, 16 for each wave,
// and 16 * VEC columns as VEC tiles, which are dealt so that a lane has VEC neighbouring
// columns of a row, a 16-byte word, and 16 lanes 256 bytes of it: tile c's column i is
// VEC * i + c.  b and h go through LDS, PRE ranks at a time, b's rows in the tiles' order.
// (6504 rows of 28672 columns, rank 32: lanes by rows as above for few 220 us, so 185, with
// registers for four blocks a CU 170, without spills, which h's shares in flight took, 153;
// for five it spills, 373.  A wave that keeps its
// columns of b and goes through the rows, their loads a round ahead, has too few of
// them on their way: 243 to 345.)
template <typename T, int PRE, bool WORDS, bool OUT_WORDS>
__global__ __launch_bounds__(256, PRE == 32 ? 4 : 3) void adapter_up_kernel(
    T* out, const T* y, const float* __restrict__ h, const T* __restrict__ b,
    const float* __restrict__ scale, const int* __restrict__ ranks,
    const int* __restrict__ plan, const Shape z, int cols) {
  using O = Operand<T>;
  constexpr int VEC = 16 / (int)sizeof(T), COLS = 16 * VEC, PITCH = PRE + VEC;
  constexpr int GRAN = PRE / VEC;                 // 16-byte words of a row in LDS
  struct alignas(16) Word { T v[VEC]; };
  __shared__ __attribute__((aligned(16))) T bs[COLS][PITCH], hs[PARTS<T>][64][PITCH];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int l15 = lane & 15, lhi = lane >> 4;
  const Place at(z, cols, COLS);
  const int place = at.tile * 64, mine = wid * 16 + lhi * 4;   // this lane's first row
  const i32x4_t own = *reinterpret_cast<const i32x4_t*>(
      plan + PLAN_HEAD + 4 * z.most + place + mine);
  const int some = (plan + PLAN_HEAD + 4 * z.most)[place];
  const i32x4_t t = reinterpret_cast<const i32x4_t*>(plan + PLAN_HEAD)[at.tile];
  const int slot = t[0], rows = t[1];
  if (at.tile >= plan[0] || (slot < 0 && out == y)) return;
  const int rank = slot < 0 ? 0 : ranks ? min(max(ranks[slot], 0), z.rank) : z.rank;
  const int n0 = at.n0, end = at.end;
  const float s = slot < 0 ? 0.f : scale[slot];
  const bool whole = OUT_WORDS && n0 + COLS <= end;
  int row[4];
  Word yv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = mine + i < rows ? own[i] : some;
  constexpr int NB = COLS * GRAN / 256;           // words of b that a thread brings
  constexpr int NH = 64 * PRE / 4 / 256;
  const long share = (long)z.T * z.parts * z.rank16;
  const T* bb = b + ((long)max(slot, 0) * z.N + n0) * z.rank;
  const float* hh = h + ((long)t[2] * z.parts + at.part) * z.rank16;
  i32x4_t bv[NB];
  f32x4_t hv[NH];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {                // columns past the part: its last
      const int g = threadIdx.x + i * 256, n = g / GRAN, j = j0 + g % GRAN * VEC;
      bv[i] = load_some<T, WORDS>(bb + (uint32_t)(min(n, end - n0 - 1) * z.rank + j),
                                  rank - j);
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const int g = threadIdx.x + i * 256, r = g / (PRE / 4), j = j0 + g % (PRE / 4) * 4;
      hv[i] = {0.f, 0.f, 0.f, 0.f};
      if (r >= rows || j >= rank) continue;
      const float* p = hh + (uint32_t)(r * z.parts * z.rank16 + j);
      hv[i] = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll 1
      for (int w = 1; w < z.split; ++w)
        hv[i] += *reinterpret_cast<const f32x4_t*>(p + w * share);
    }
  };
  fetch(0);
  if (whole)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      yv[i] = *reinterpret_cast<const Word*>(y + (long)row[i] * z.ldy + n0 + l15 * VEC);
  if (rank == 0 && out == y) return;
  f32x4_t acc[VEC];
#pragma unroll
  for (int c = 0; c < VEC; ++c) acc[c] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int j0 = 0; j0 < rank; j0 += PRE) {
    if (j0 > 0) {
      fetch(j0);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int g = threadIdx.x + i * 256, n = g / GRAN;
      *reinterpret_cast<i32x4_t*>(&bs[n % VEC * 16 + n / VEC][g % GRAN * VEC]) = bv[i];
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const int g = threadIdx.x + i * 256, r = g / (PRE / 4), j = g % (PRE / 4) * 4;
      const Four<T> f(hv[i], s, rank - j0 - j);
#pragma unroll
      for (int p = 0; p < PARTS<T>; ++p) f.put(p, &hs[p][r][j]);
    }
    __syncthreads();
    if (wid * 16 < rows)
#pragma unroll
      for (int k = 0; k < PRE; k += O::STEP) {
        if (j0 + k >= rank) break;
        i32x4_t hw[PARTS<T>];
#pragma unroll
        for (int p = 0; p < PARTS<T>; ++p)
          hw[p] = *reinterpret_cast<const i32x4_t*>(&hs[p][wid * 16 + l15][k + lhi * O::PER]);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          const i32x4_t bw =
              *reinterpret_cast<const i32x4_t*>(&bs[c * 16 + l15][k + lhi * O::PER]);
#pragma unroll
          for (int p = 0; p < PARTS<T>; ++p) acc[c] = O::mul(hw[p], bw, acc[c]);
        }
      }
  }
  // register i of tile c: row 4 * (lane / 16) + i, column VEC * (lane % 16) + c
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (mine + i >= rows) break;
    if (whole) {
      Word w = yv[i];
      if (rank > 0)
#pragma unroll
        for (int c = 0; c < VEC; ++c) w.v[c] = (T)((float)w.v[c] + acc[c][i]);
      *reinterpret_cast<Word*>(out + (long)row[i] * z.ldo + n0 + l15 * VEC) = w;
    } else {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const int n = n0 + l15 * VEC + c;
        if (n >= end) break;
        const T old = y[(long)row[i] * z.ldy + n];
        out[(long)row[i] * z.ldo + n] = rank > 0 ? (T)((float)old + acc[c][i]) : old;
      }
    }
  }
}

// ------------------------------------------------------------------ bindings
// Rows of a tile: 16 of few rows, whose tiles would stay empty.  By rows alone: the rows of
// each adapter, which decide, are known on the device.  (us, 4096 -> 4096, 1024, 1024 bf16,
// rank 16, tiles of 16 and of 64: 4 adapters, 48, 128, 256, 257, 512, 1024 rows 9.8, 10.1, 10.7,
// 10.6, 12.4, 18.2 and 10.0, 10.2, 10.9, 11.0, 12.4, 16.1; 64 adapters 15.0, 17.8, 18.5, 18.4,
// 19.6, 21.5 and 25.8, 32.0, 33.2, 33.0, 34.6, 38.7; 512 adapters 15.0, 25.4, 50, 56, 93, 94 and
// 25.5, 53.6, 113, 116, 217, 225.  So beyond the line many adapters would do better in 16.)
static int tile_rows(long T) { return T <= 256 ? 16 : 64; }
static long most_tiles(long T, long slots) {
  return T / tile_rows(T) + std::min(T, slots + 1);
}

torch::Tensor adapter_plan(torch::Tensor index, int64_t slots) {
  TORCH_CHECK(index.is_cuda() && index.dim() == 1 && index.is_contiguous() &&
                  index.scalar_type() == torch::kInt32 && index.numel() < (1L << 24),
              "adapter_plan: index (T) int32 on the GPU");
  TORCH_CHECK(slots >= 1 && slots <= MOST_SLOTS, "adapter_plan: 1 to ", MOST_SLOTS,
              " adapters");
  const c10::DeviceGuard guard(index.device());
  const long T = index.numel(), most = most_tiles(T, slots);
  auto plan = torch::empty({PLAN_HEAD + (4 + tile_rows(T)) * most}, index.options());
  if (T == 0) return plan;
  adapter_plan_kernel<<<dim3(1), dim3(1024), 0, at::hip::getCurrentHIPStream()>>>(
      plan.data_ptr<int>(), index.data_ptr<int>(), (int)T, (int)slots, tile_rows(T),
      (int)most);
  HIP_CHECK_KERNEL();
  return plan;
}

template <typename T>
static void launch_adapter_add(torch::Tensor& out, const torch::Tensor& y,
                               const torch::Tensor& x, const torch::Tensor& a,
                               const torch::Tensor& b, const torch::Tensor& scale,
                               const int* ranks, const torch::Tensor& plan, Shape z,
                               bool words_down, bool words_up, bool words_out) {
  auto stream = at::hip::getCurrentHIPStream();
  const int* pl = plan.data_ptr<int>();
  // Up to 1024 rows a block takes 16 of them in 16 waves, else 32 in 4: of few rows there
  // are too few blocks otherwise, of many each one reads A again (620 rows, fp32, 8960 -> 20
  // 21 us in blocks of 32 rows and 16 of 16; 6504 rows, bf16, 14336 -> 32, before the
  // loads were dealt as they are, 72 and 97; since then, four projections of those rows, 132
  // in blocks of 8 waves and 125 of 4).  Around the line, both products, as at tile_rows:
  // 4 adapters, 512, 1024, 1500, 2048, 4096 rows 12.4, 16.2, 23.3, 23.3, 38.8 in blocks of 16
  // rows and 15.1, 18.4, 23.2, 26.8, 38.2 of 32; 64 adapters 34.7, 38.1, 40.9, 42.2, 52.9 and
  // 25.1, 26.8, 29.2, 31.0, 39.3.
  const int sixteens = tile_rows(z.T) / 16, RT = z.T <= 1024 ? 1 : 2, NW = RT == 1 ? 16 : 4;
  const int subs = sixteens / RT;
  // Tiles of ranks that a block takes: all of them in equal groups, of up to two where a wave
  // of 16 has 128 registers (three spill: 128 rows, 3 x 16 ranks of 4096, 8.0 us and 6.5 by
  // two; 57 rows, 3 x 64 ranks of 3584 16.2 and 19.2, 2 x 64 15.0 and 11.8), of up to four
  // where it has twice as many and reads x for each group
  const int tiles = z.rank16 / 16 * z.parts, most_ct = RT == 1 ? 2 : 4;
  const int groups = (tiles + most_ct - 1) / most_ct, CT = (tiles + groups - 1) / groups;
  const long blocks = (long)z.most * subs * ((tiles + CT - 1) / CT);
  // shares of the inner dimension until there are 512 blocks, each wave with a round at
  // least; no more than up to four, because up adds them in every block
  z.split = (int)std::max<long>(
      1, std::min<long>({512 / blocks, (long)z.K * y.element_size() / (NW * 256),
                         MOST_SPLIT}));
  auto h = torch::empty({(long)z.split * z.T * z.parts * z.rank16},
                        y.options().dtype(torch::kFloat32));
  TORCH_CHECK(blocks * z.split < (1L << 31), "adapter_add: too many rows");
  auto down = [&](auto kern, int waves) {
    kern<<<dim3((unsigned)(blocks * z.split)), dim3(waves * 64), 0, stream>>>(
        h.data_ptr<float>(), (const T*)x.data_ptr(), (const T*)a.data_ptr(), ranks, pl, z,
        subs);
  };
#define DOWN(N, R, C, W)                                         \
  if (RT == R && CT == C && words_down == W)                     \
    down(adapter_down_kernel<T, N, R, C, W>, N);
#define DOWNS(N, R, C) DOWN(N, R, C, true) DOWN(N, R, C, false)
  DOWNS(16, 1, 1) DOWNS(16, 1, 2)
  DOWNS(4, 2, 1) DOWNS(4, 2, 2) DOWNS(4, 2, 3) DOWNS(4, 2, 4)
#undef DOWNS
#undef DOWN
  HIP_CHECK_KERNEL();
  const int wide = sixteens == 1 ? FEW_COLS : 16 * 16 / (int)sizeof(T);
  int cols = 0;
  for (int p = 0; p < z.parts; ++p)
    cols += (z.first[p + 1] - z.first[p] + wide - 1) / wide;
  TORCH_CHECK((long)z.most * cols < (1L << 31), "adapter_add: too many rows");
  auto up = [&](auto kern) {
    kern<<<dim3((unsigned)((long)z.most * cols)), dim3(256), 0, stream>>>(
        (T*)out.data_ptr(), (const T*)y.data_ptr(), h.data_ptr<float>(),
        (const T*)b.data_ptr(), scale.data_ptr<float>(), ranks, pl, z, cols);
  };
#define UP(W, O)                                                        \
  if (words_up == W && words_out == O) {                                \
    if (sixteens == 1) up(adapter_up_few_kernel<T, W, O>);              \
    else if (z.rank <= 32) up(adapter_up_kernel<T, 32, W, O>);          \
    else up(adapter_up_kernel<T, 64, W, O>);                            \
  }
  UP(true, true) UP(true, false) UP(false, true) UP(false, false)
#undef UP
  HIP_CHECK_KERNEL();
}

torch::Tensor adapter_add(const torch::Tensor& y, const torch::Tensor& x,
                          const torch::Tensor& a, const torch::Tensor& b,
                          const torch::Tensor& scale,
                          const c10::optional<torch::Tensor>& ranks,
                          const torch::Tensor& plan, int64_t rows, int64_t slots,
                          std::vector<int64_t> widths,
                          const c10::optional<torch::Tensor>& into) {
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(y.requires_grad() || x.requires_grad() || a.requires_grad() ||
                    b.requires_grad() || scale.requires_grad() ||
                    (into.has_value() && into->requires_grad())),
              "adapter_add has no gradients: call it under torch.no_grad()");
  torch::Tensor out = into.has_value() ? *into : torch::empty(y.sizes(), y.options());
  if (widths.empty() && y.dim() == 2) widths.push_back(y.size(1));
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && x.dim() == 2 && a.dim() == 4 &&
                  b.dim() == 3 && out.sizes() == y.sizes(),
              "adapter_add: y, out (T, N), x (T, K), a (S, P, r, K), b (S, N, r)");
  const long T = y.size(0), N = y.size(1), K = x.size(1), S = a.size(0), r = a.size(2);
  TORCH_CHECK(x.size(0) == T && a.size(3) == K && a.size(1) == (long)widths.size() &&
                  b.size(0) == S && b.size(1) == N && b.size(2) == r && S == slots,
              "adapter_add: shapes that do not fit together");
  TORCH_CHECK(widths.size() >= 1 && widths.size() <= 8 && r >= 1 && r <= MOST_RANK &&
                  K >= 1 && K < (1L << 20) && N < (1L << 30),
              "adapter_add: 1 to 8 parts, ranks 1 to ", MOST_RANK, ", inner widths below 2^20");
  for (const auto& t : {out, x, a, b})
    TORCH_CHECK(t.device() == y.device() && t.scalar_type() == y.scalar_type(),
                "adapter_add: tensors of one type and device");
  for (const auto& t : {out, y, x})
    TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, "adapter_add: rows of adjacent numbers");
  TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "adapter_add: contiguous a and b");
  TORCH_CHECK(T <= 1 || out.stride(0) >= N,
              "adapter_add: out is y or apart from it, its rows from each other");
  if (into.has_value()) {
    const bool in_place = out.data_ptr() == y.data_ptr() && out.strides() == y.strides();
    TORCH_CHECK(in_place || !rows_overlap(out, y),
                "adapter_add: out is y or apart from it, its rows from each other");
    for (const auto& t : {x, a, b})
      TORCH_CHECK(!rows_overlap(out, t), "adapter_add: out on top of an operand");
  }
  TORCH_CHECK(scale.device() == y.device() && scale.scalar_type() == torch::kFloat32 &&
                  scale.is_contiguous() && scale.numel() == S,
              "adapter_add: scale (S) fp32");
  const bool some = ranks.has_value();
  TORCH_CHECK(!some || (ranks->device() == y.device() && ranks->is_contiguous() &&
                        ranks->scalar_type() == torch::kInt32 && ranks->numel() == S),
              "adapter_add: ranks (S) int32");
  Shape z{};
  z.T = (int)T, z.K = (int)K, z.N = (int)N, z.parts = (int)widths.size();
  z.rank = (int)r, z.rank16 = (int)((r + 15) / 16 * 16);
  z.ldx = x.stride(0), z.ldy = y.stride(0), z.ldo = out.stride(0);
  z.most = (int)most_tiles(T, S);
  TORCH_CHECK(plan.device() == y.device() && plan.scalar_type() == torch::kInt32 &&
                  rows == T && plan.numel() == PLAN_HEAD + (4L + tile_rows(T)) * z.most,
              "adapter_add: a plan of other rows");
  const long size = y.element_size();
  auto whole = [&](const torch::Tensor& t, long row) {
    return ((uintptr_t)t.data_ptr() & 15) == 0 && row * size % 16 == 0;
  };
  bool words_out = whole(out, z.ldo) && whole(y, z.ldy);
  long left = N;
  for (size_t p = 0; p < widths.size(); ++p) {
    TORCH_CHECK(widths[p] >= 0 && widths[p] <= left,
                "adapter_add: widths that do not add up to N");
    left -= widths[p];
    words_out = words_out && z.first[p] * size % 16 == 0;
    z.first[p + 1] = z.first[p] + (int)widths[p];
  }
  TORCH_CHECK(left == 0, "adapter_add: widths that do not add up to N");
  if (T == 0 || N == 0) return out;
  const bool words_down = whole(x, z.ldx) && whole(a, K), words_up = whole(b, r);
  const c10::DeviceGuard guard(y.device());
  const int* rk = some ? ranks->data_ptr<int>() : nullptr;
  if (y.scalar_type() == torch::kBFloat16)
    launch_adapter_add<__bf16>(out, y, x, a, b, scale, rk, plan, z, words_down, words_up,
                       words_out);
  else if (y.scalar_type() == torch::kFloat32)
    launch_adapter_add<float>(out, y, x, a, b, scale, rk, plan, z, words_down, words_up,
                       words_out);
  else
    TORCH_CHECK(false, "adapter_add: dtype must be bf16 or fp32");
  if (into.has_value()) written(out);
  return out;
}
