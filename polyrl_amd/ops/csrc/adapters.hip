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
// and adds the result to y, which it reads and writes once.
//
// Matrix cores: 16x16x32 in bf16, 16x16x4 in fp32.  h is a sum in 32 bits; as an operand
// in bf16 it is split in two bf16 numbers, h = hi + lo, each with its own product, so that what
// is lost of it is 2^-16 and not the 2^-8 of one.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"

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
// plan: tiles, then (4 ints each) adapter, first place, rows; then the rows by place.
// Rows without an adapter come last, as tiles of adapter -1.
constexpr int PLAN_HEAD = 4;
constexpr int MOST_SLOTS = 4095;

__global__ __launch_bounds__(1024) void adapter_plan_kernel(int* plan, const int* index,
                                                            int T, int slots, int tile,
                                                            int most) {
  __shared__ int count[MOST_SLOTS + 1], cursor[MOST_SLOTS + 1];
  __shared__ int sum_rows[1024], sum_tiles[1024];
  const int tid = threadIdx.x;
  for (int s = tid; s <= slots; s += 1024) count[s] = 0;
  __syncthreads();
  // rows of the wave's first row's adapter are counted by one lane, twice; a prompt's
  // are all of them
  for (int t0 = 0; t0 < T; t0 += 1024) {
    const int t = t0 + tid;
    int s = t < T ? index[t] : -2;
    if (t < T && (s < 0 || s >= slots)) s = slots;
    bool mine = s >= 0;
    for (int r = 0; r < 2; ++r) {
      const unsigned long long left = __ballot(mine);
      if (left == 0) break;
      const int first = __ffsll(left) - 1;
      const int f = __shfl(s, first, 64);
      const unsigned long long same = __ballot(mine && s == f);
      if ((tid & 63) == first) atomicAdd(&count[f], __popcll(same));
      if (s == f) mine = false;
    }
    if (mine) atomicAdd(&count[s], 1);
  }
  __syncthreads();
  // each thread a stretch of adapters, then the stretches' sums
  const int per = (slots + 1 + 1023) / 1024;
  int rows = 0, tiles = 0;
  for (int s = tid * per; s < min((tid + 1) * per, slots + 1); ++s) {
    rows += count[s];
    tiles += (count[s] + tile - 1) / tile;
  }
  sum_rows[tid] = rows;
  sum_tiles[tid] = tiles;
  __syncthreads();
  for (int d = 1; d < 1024; d *= 2) {
    const int r = tid >= d ? sum_rows[tid - d] : 0;
    const int n = tid >= d ? sum_tiles[tid - d] : 0;
    __syncthreads();
    sum_rows[tid] += r;
    sum_tiles[tid] += n;
    __syncthreads();
  }
  if (tid == 1023) plan[0] = sum_tiles[1023];
  i32x4_t* entry = reinterpret_cast<i32x4_t*>(plan + PLAN_HEAD);
  int at = sum_rows[tid] - rows, n = sum_tiles[tid] - tiles;
  for (int s = tid * per; s < min((tid + 1) * per, slots + 1); ++s) {
    cursor[s] = at;
    for (int i = 0; i < count[s]; i += tile, ++n)
      entry[n] = i32x4_t{s < slots ? s : -1, at + i, min(tile, count[s] - i), 0};
    at += count[s];
  }
  __syncthreads();
  int* order = plan + PLAN_HEAD + 4 * most;
  for (int t0 = 0; t0 < T; t0 += 1024) {
    const int t = t0 + tid;
    int s = t < T ? index[t] : -2;
    if (t < T && (s < 0 || s >= slots)) s = slots;
    bool mine = s >= 0;
    for (int r = 0; r < 2; ++r) {
      const unsigned long long left = __ballot(mine);
      if (left == 0) break;
      const int first = __ffsll(left) - 1;
      const int f = __shfl(s, first, 64);
      const bool now = mine && s == f;
      const unsigned long long same = __ballot(now);
      int place = 0;
      if ((tid & 63) == first) place = atomicAdd(&cursor[f], __popcll(same));
      place = __shfl(place, first, 64);
      if (now) {
        order[place + __popcll(same & ((1ull << (tid & 63)) - 1))] = t;
        mine = false;
      }
    }
    if (mine) order[atomicAdd(&cursor[s], 1)] = t;
  }
}

// ---------------------------------------------------------------------- down
struct Shape {
  int T, K, N, parts, rank, rank16;   // rank16: rank rounded up to whole tiles of 16
  long ldx, ldy, ldo;
  int split, most;
  int first[9];                       // columns of the parts
};

// h[share][place][part][j], one block a tile of rows, CT tiles of ranks of a part and a
// share of the inner dimension
template <typename T, int RT, int CT, bool WORDS>
__global__ __launch_bounds__(256) void adapter_down_kernel(
    float* __restrict__ h, const T* __restrict__ x, const T* __restrict__ a,
    const int* __restrict__ ranks, const int* __restrict__ plan, const Shape z) {
  using O = Operand<T>;
  __shared__ float red[4 * RT * CT * 256];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int l15 = lane & 15, lhi = lane >> 4;
  const int groups = (z.rank16 / 16 + CT - 1) / CT;
  int id = blockIdx.x;
  const int share = id % z.split;
  id /= z.split;
  const int group = id % groups;
  id /= groups;
  const int part = id % z.parts, tile = id / z.parts;
  if (tile >= plan[0]) return;
  const i32x4_t t = reinterpret_cast<const i32x4_t*>(plan + PLAN_HEAD)[tile];
  const int slot = t[0], place = t[1], rows = t[2];
  if (slot < 0) return;
  const int rank = ranks ? min(max(ranks[slot], 0), z.rank) : z.rank;
  const int j0 = group * CT * 16;
  if (j0 >= rank) return;
  const int* order = plan + PLAN_HEAD + 4 * z.most + place;
  // this wave's share of the inner dimension, in whole lines of 128 bytes
  const int line = 128 / (int)sizeof(T), lines = (z.K + line - 1) / line;
  const int per = (lines + z.split * 4 - 1) / (z.split * 4) * line;
  const int k0 = (share * 4 + wid) * per, k1 = min(k0 + per, z.K);
  const T* xr[RT];
  const T* ar[CT];
#pragma unroll
  for (int r = 0; r < RT; ++r)        // rows past the tile: any, dropped below
    xr[r] = x + (long)order[min(r * 16 + l15, rows - 1)] * z.ldx + lhi * O::PER;
#pragma unroll
  for (int c = 0; c < CT; ++c)
    ar[c] = a + (((long)slot * z.parts + part) * z.rank +
                 min(j0 + c * 16 + l15, rank - 1)) * z.K + lhi * O::PER;
  f32x4_t acc[RT][CT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[r][c] = {0.f, 0.f, 0.f, 0.f};
  for (int k = k0; k < k1; k += O::STEP) {
    const int have = k1 - k - lhi * O::PER;
    i32x4_t xv[RT], av[CT];
#pragma unroll
    for (int r = 0; r < RT; ++r) xv[r] = load_some<T, WORDS>(xr[r] + k, have);
#pragma unroll
    for (int c = 0; c < CT; ++c) av[c] = load_some<T, WORDS>(ar[c] + k, have);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[r][c] = O::mul(xv[r], av[c], acc[r][c]);
  }
  // sums of the four waves; register i: row 4 * (lane / 16) + i, column lane % 16
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[((wid * RT + r) * CT + c) * 256 + (lhi * 4 + i) * 16 + l15] = acc[r][c][i];
  __syncthreads();
  const int row = threadIdx.x / 16, col = threadIdx.x % 16;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        v += red[((w * RT + r) * CT + c) * 256 + threadIdx.x];
      const int j = j0 + c * 16 + col;
      if (r * 16 + row < rows && j < rank)
        h[(((long)share * z.T + place + r * 16 + row) * z.parts + part) * z.rank16 + j] = v;
    }
}

// ------------------------------------------------------------------------ up
// A block takes a tile of rows and 256 columns of one part, a wave 64 of them as four
// tiles of 16, which are dealt so that a lane holds 16 neighbouring columns of its row:
// tile c's row i is column 16 * (i / 4) + 4 * c + i % 4.
constexpr int UP_COLS = 256, UP_RANK = 64;

// WORDS: rows of b come in whole 16-byte words; OUT_WORDS: those of y and out
template <typename T, int RT, bool WORDS, bool OUT_WORDS>
__global__ __launch_bounds__(256) void adapter_up_kernel(
    T* out, const T* y, const float* __restrict__ h, const T* __restrict__ b,
    const float* __restrict__ scale, const int* __restrict__ ranks,
    const int* __restrict__ plan, const Shape z, int cols) {
  using O = Operand<T>;
  constexpr bool SPLIT = sizeof(T) == 2;          // h as hi + lo
  constexpr int PITCH = UP_RANK + 16 / (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) T hs[SPLIT ? 2 : 1][RT * 16][PITCH];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int l15 = lane & 15, lhi = lane >> 4;
  const int tile = blockIdx.x / cols;
  int col = blockIdx.x % cols, part = 0;
  if (tile >= plan[0]) return;
  while (col >= (z.first[part + 1] - z.first[part] + UP_COLS - 1) / UP_COLS) {
    col -= (z.first[part + 1] - z.first[part] + UP_COLS - 1) / UP_COLS;
    ++part;
  }
  const i32x4_t t = reinterpret_cast<const i32x4_t*>(plan + PLAN_HEAD)[tile];
  const int slot = t[0], place = t[1], rows = t[2];
  const int rank = slot < 0 ? 0 : ranks ? min(max(ranks[slot], 0), z.rank) : z.rank;
  if (rank == 0 && out == y) return;
  const int* order = plan + PLAN_HEAD + 4 * z.most + place;
  const int end = z.first[part + 1];
  const int n0 = z.first[part] + col * UP_COLS + wid * 64;
  const float s = slot < 0 ? 0.f : scale[slot];
  f32x4_t acc[RT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[r][c] = {0.f, 0.f, 0.f, 0.f};
  const T* br[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)                     // columns past the part: its last
    br[c] = b + ((long)max(slot, 0) * z.N +
                 min(n0 + l15 / 4 * 16 + c * 4 + l15 % 4, end - 1)) * z.rank +
            lhi * O::PER;
  for (int j0 = 0; j0 < rank; j0 += UP_RANK) {
    const int have = min(rank - j0, UP_RANK);
    if (j0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < RT * 16 * UP_RANK; i += 256) {
      const int r = i / UP_RANK, j = i % UP_RANK;
      float v = 0.f;
      if (r < rows && j < have) {
        const float* p = h + (((long)place + r) * z.parts + part) * z.rank16 + j0 + j;
        for (int w = 0; w < z.split; ++w)
          v += p[(long)w * z.T * z.parts * z.rank16];
        v *= s;
      }
      const T hi = (T)v;
      hs[0][r][j] = hi;
      // (an infinite h has no lower part)
      if (SPLIT) hs[SPLIT ? 1 : 0][r][j] = isfinite((float)hi) ? (T)(v - (float)hi) : (T)0.f;
    }
    __syncthreads();
    for (int k = 0; k < have; k += O::STEP) {
      i32x4_t bv[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        bv[c] = load_some<T, WORDS>(br[c] + j0 + k, have - k - lhi * O::PER);
#pragma unroll
      for (int p = 0; p < (SPLIT ? 2 : 1); ++p)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const i32x4_t hv = *reinterpret_cast<const i32x4_t*>(
              &hs[p][r * 16 + l15][k + lhi * O::PER]);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[r][c] = O::mul(bv[c], hv, acc[r][c]);
        }
    }
  }
  // lane: row lane % 16 of every 16, columns 16 * (lane / 16) .. + 16
  const int n = n0 + lhi * 16;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    if (r * 16 + l15 >= rows) continue;
    const long row = order[r * 16 + l15];
    const T* from = y + row * z.ldy + n;
    T* to = out + row * z.ldo + n;
    struct alignas(16) Word { T v[16 / sizeof(T)]; };
    constexpr int VEC = 16 / (int)sizeof(T);
    if (OUT_WORDS && n + 16 <= end) {
#pragma unroll
      for (int q = 0; q < 16 / VEC; ++q) {
        Word w = reinterpret_cast<const Word*>(from)[q];
        if (rank > 0) {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            w.v[i] = (T)((float)w.v[i] + acc[r][(q * VEC + i) / 4][(q * VEC + i) % 4]);
        }
        reinterpret_cast<Word*>(to)[q] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (n + i < end)
          to[i] = rank > 0 ? (T)((float)from[i] + acc[r][i / 4][i % 4]) : from[i];
    }
  }
}

// ------------------------------------------------------------------ bindings
// rows of a tile: 16 of few rows, whose tiles would stay empty
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
  auto plan = torch::empty({PLAN_HEAD + 4 * most + T}, index.options());
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
  const int RT = tile_rows(z.T) / 16, tiles16 = z.rank16 / 16;
  const int CT = tiles16 >= 3 ? 4 : tiles16;
  const int groups = (tiles16 + CT - 1) / CT;
  const long blocks = (long)z.most * z.parts * groups;
  z.split = (int)std::max<long>(1, std::min<long>({768 / blocks, z.K / 256, 16}));
  auto h = torch::empty({(long)z.split * z.T * z.parts * z.rank16},
                        y.options().dtype(torch::kFloat32));
  TORCH_CHECK(blocks * z.split < (1L << 31), "adapter_add: too many rows");
  auto down = [&](auto kern) {
    kern<<<dim3((unsigned)(blocks * z.split)), dim3(256), 0, stream>>>(
        h.data_ptr<float>(), (const T*)x.data_ptr(), (const T*)a.data_ptr(), ranks, pl, z);
  };
#define DOWN(R, C)                                          \
  if (RT == R && CT == C) {                                 \
    words_down ? down(adapter_down_kernel<T, R, C, true>)   \
               : down(adapter_down_kernel<T, R, C, false>); \
  }
  DOWN(1, 1) DOWN(1, 2) DOWN(1, 4) DOWN(4, 1) DOWN(4, 2) DOWN(4, 4)
#undef DOWN
  HIP_CHECK_KERNEL();
  int cols = 0;
  for (int p = 0; p < z.parts; ++p)
    cols += (z.first[p + 1] - z.first[p] + UP_COLS - 1) / UP_COLS;
  TORCH_CHECK((long)z.most * cols < (1L << 31), "adapter_add: too many rows");
  auto up = [&](auto kern) {
    kern<<<dim3((unsigned)((long)z.most * cols)), dim3(256), 0, stream>>>(
        (T*)out.data_ptr(), (const T*)y.data_ptr(), h.data_ptr<float>(),
        (const T*)b.data_ptr(), scale.data_ptr<float>(), ranks, pl, z, cols);
  };
#define UP(R, W, O) \
  if (RT == R && words_up == W && words_out == O) up(adapter_up_kernel<T, R, W, O>);
  UP(1, true, true) UP(1, true, false) UP(1, false, true) UP(1, false, false)
  UP(4, true, true) UP(4, true, false) UP(4, false, true) UP(4, false, false)
#undef UP
  HIP_CHECK_KERNEL();
}

void adapter_add(torch::Tensor out, torch::Tensor y, torch::Tensor x, torch::Tensor a,
                 torch::Tensor b, torch::Tensor scale, torch::Tensor ranks,
                 torch::Tensor plan, int64_t slots, std::vector<int64_t> widths) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && x.dim() == 2 && a.dim() == 4 &&
                  b.dim() == 3 && out.sizes() == y.sizes(),
              "adapter_add: y, out (T, N), x (T, K), a (S, P, r, K), b (S, N, r)");
  const long T = y.size(0), N = y.size(1), K = x.size(1), S = a.size(0), r = a.size(2);
  TORCH_CHECK(x.size(0) == T && a.size(3) == K && a.size(1) == (long)widths.size() &&
                  b.size(0) == S && b.size(1) == N && b.size(2) == r && S == slots,
              "adapter_add: shapes that do not fit together");
  TORCH_CHECK(widths.size() >= 1 && widths.size() <= 8 && r >= 1 && r <= 4096 &&
                  K >= 1 && K < (1L << 30) && N < (1L << 30),
              "adapter_add: 1 to 8 parts, ranks 1 to 4096");
  for (const auto& t : {out, x, a, b})
    TORCH_CHECK(t.device() == y.device() && t.scalar_type() == y.scalar_type(),
                "adapter_add: tensors of one type and device");
  for (const auto& t : {out, y, x})
    TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, "adapter_add: rows of adjacent numbers");
  TORCH_CHECK(out.data_ptr() != y.data_ptr() || out.strides() == y.strides(),
              "adapter_add: out is y or apart from it");
  TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "adapter_add: contiguous a and b");
  TORCH_CHECK(scale.device() == y.device() && scale.scalar_type() == torch::kFloat32 &&
                  scale.is_contiguous() && scale.numel() == S,
              "adapter_add: scale (S) fp32");
  const bool some = ranks.defined() && ranks.numel() > 0;
  TORCH_CHECK(!some || (ranks.device() == y.device() && ranks.is_contiguous() &&
                        ranks.scalar_type() == torch::kInt32 && ranks.numel() == S),
              "adapter_add: ranks (S) int32");
  Shape z{};
  z.T = (int)T, z.K = (int)K, z.N = (int)N, z.parts = (int)widths.size();
  z.rank = (int)r, z.rank16 = (int)((r + 15) / 16 * 16);
  z.ldx = x.stride(0), z.ldy = y.stride(0), z.ldo = out.stride(0);
  z.most = (int)most_tiles(T, S);
  TORCH_CHECK(plan.device() == y.device() && plan.scalar_type() == torch::kInt32 &&
                  plan.numel() == PLAN_HEAD + 4L * z.most + T,
              "adapter_add: a plan of other rows");
  const long size = y.element_size();
  auto whole = [&](const torch::Tensor& t, long row) {
    return ((uintptr_t)t.data_ptr() & 15) == 0 && row * size % 16 == 0;
  };
  bool words_out = whole(out, z.ldo) && whole(y, z.ldy);
  for (size_t p = 0; p < widths.size(); ++p) {
    TORCH_CHECK(widths[p] >= 0 && widths[p] <= N, "adapter_add: widths of the parts");
    words_out = words_out && z.first[p] * size % 16 == 0;
    z.first[p + 1] = z.first[p] + (int)widths[p];
  }
  TORCH_CHECK(z.first[widths.size()] == N, "adapter_add: widths that do not add up to N");
  if (T == 0 || N == 0) return;
  const bool words_down = whole(x, z.ldx) && whole(a, K), words_up = whole(b, r);
  const c10::DeviceGuard guard(y.device());
  const int* rk = some ? ranks.data_ptr<int>() : nullptr;
  if (y.scalar_type() == torch::kBFloat16)
    launch_adapter_add<__bf16>(out, y, x, a, b, scale, rk, plan, z, words_down, words_up,
                       words_out);
  else if (y.scalar_type() == torch::kFloat32)
    launch_adapter_add<float>(out, y, x, a, b, scale, rk, plan, z, words_down, words_up,
                       words_out);
  else
    TORCH_CHECK(false, "adapter_add: dtype must be bf16 or fp32");
}
