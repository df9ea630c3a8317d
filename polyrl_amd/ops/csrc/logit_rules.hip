// Rules of a request on its next token's logits, and the tokens that they go by.
//
//   u   = seen in prompt or output ? (l > 0 ? l / repetition : l * repetition) : l
//   out = allowed ? u - frequency * c - presence * [c > 0] + bias : -inf
// with c the token's times in the output so far.  Computed in 32 bits, rounded once to
// the logits' type.
//
// Split.  No table of counts is kept per request (a row of 128256 would be as long as
// its logits, read at every token and copied with every fork): the history itself is the
// state.  A block takes a chunk of one row, counts the part of the history that falls into
// it in LDS (a word per token: times said, seen, its bias), and passes over the logits once.
//
// What bounds it: memory, and before it the chain row -> slot -> history -> counts in each
// block (128 x 128256 bf16, 257 to 512 tokens of history, 16 biases: 17.0 us, 3.9 TB/s, 12
// without rules; 64 x 151936 fp32 with masks 17.6, 4.5 TB/s, what a copy takes).  Long
// histories are read by every chunk of their row, which waits for each round of them but the
// first (33 x 152064, 9000 to 32768 tokens: 18.6).
// What it took: 4-byte reads of the history, one waited for after the other 54 us of the
// last, words 33; loads of the logits behind those of the history, so that a wait for
// these does not wait for them, and barriers for LDS alone 19.9 -> 18.1 of the first; blocks of
// 256 threads or chunks of four words a thread 20 to 24.  Bits for the tokens that the
// counts touch, whose words alone are cleared, lose (20.5; 24.1 for 16.9 of the last).
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "rows_overlap.h"
#include "vocab_row.h"

typedef __attribute__((ext_vector_type(4))) int i32x4_t;

// a token's word in LDS
constexpr uint32_t SAID = (1u << 19) - 1;   // times in the output
constexpr uint32_t SEEN = 1u << 19;         // in the prompt
constexpr int BIAS = 20;                    // from here: place in the biases + 1
constexpr long MOST_TOKENS = SAID, MOST_BIASES = (1 << 12) - 1;

struct Rules {
  const int* rows;
  const int* history;
  const int* prompt_len;
  const int* total_len;
  const float *repetition, *frequency, *presence;
  const int* bias_tokens;
  const float* bias_values;
  const int* mask;
  const int* masked;
  int slots, cap, biases, words;
};

// one rounding for each operation: the sums are the definition's
DEV_INLINE float ruled(float l, uint32_t w, float rep, float freq, float pres,
                       const float* __restrict__ values) {
  const uint32_t c = w & SAID;
  if (w & (SAID | SEEN)) l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
  if (c) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)c)), pres);
  if (w >> BIAS) l = __fadd_rn(l, values[(w >> BIAS) - 1]);
  return l;
}

template <typename T> DEV_INLINE T rounded(float x);
template <> DEV_INLINE float rounded<float>(float x) { return x; }
template <> DEV_INLINE bf16_t rounded<bf16_t>(float x) { return f2bf(x); }

constexpr int NT = 512;                     // threads of a block
constexpr int HW = 2;                       // words of history that a thread has at a time

// A barrier for what lies in LDS alone: loads from memory stay on their way
DEV_INLINE void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A block takes NT * U words of VEC tokens of a row, each thread U of them, which are on
// their way while the history is counted.  WIDE: a row of logits and its row of out start
// at the same place of a 16-byte word
template <typename T, bool WIDE, int U>
__global__ __launch_bounds__(NT) void logit_rules_kernel(
    T* out, const T* logits, const Rules a, int V, long ld, long ld_out, int chunks) {
  constexpr int VEC = WIDE ? VocabRow<T>::VEC : 1, CHUNK = NT * U * VEC;
  struct alignas(VEC * sizeof(T)) Word { T v[VEC]; };
  __shared__ __attribute__((aligned(16))) uint32_t lds[CHUNK];
  const long row = blockIdx.x / chunks;
  const int part = blockIdx.x % chunks, tid = threadIdx.x;
  const VocabRow<T> in(logits + row * ld, V);
  T* to = out + row * ld_out;
  // groups of VEC tokens; the first one of a row that starts inside a word is short
  const int lead = WIDE ? in.lead : 0, ahead = WIDE ? 1 : 0;
  const int g0 = part * NT * U;
  const int base = lead + (g0 - ahead) * VEC;     // the chunk's first token, may be < 0
  // LDS word of the chunk's token t: a thread's VEC tokens in two halves (of 8), so that
  // neighbours read neighbouring 16-byte words
  auto at = [](int t) {
    return VEC == 8 ? t / 8 * 4 + t % 4 + (t & 4) * (CHUNK / 8) : t;
  };
  const bool same = out == logits;
  Word v[U];
  auto load = [&](int u) {
    const int i0 = base + (u * NT + tid) * VEC;
    if (i0 >= 0 && i0 + VEC <= V) {
      v[u] = *reinterpret_cast<const Word*>(in.x + i0);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (i0 + j >= 0 && i0 + j < V) v[u].v[j] = in.x[i0 + j];
    }
  };
  const int slot = a.rows[row];
  float rep = 1.f, freq = 0.f, pres = 0.f;
  bool counts = false, biased = false, masked = false;
  int total = 0, prompt = 0;
  if (slot >= 0 && slot < a.slots) {
    rep = a.repetition[slot], freq = a.frequency[slot], pres = a.presence[slot];
    total = min(max(a.total_len[slot], 0), a.cap);
    prompt = min(max(a.prompt_len[slot], 0), total);
    counts = total > 0 && (rep != 1.f || freq != 0.f || pres != 0.f);
    biased = a.biases > 0;
    masked = a.masked[slot] != 0;
  }
  if (same && !counts && !biased && !masked) return;
  // What is read is on its way in the order in which it is needed, the logits last: they
  // arrive while the history is counted.
  const int* h = a.history + (long)slot * a.cap;
  const int head = min((int)((16 - ((uintptr_t)h & 15)) & 15) / 4, total);
  const int whole = counts ? (total - head) / 4 : 0, tail = head + whole * 4;
  const i32x4_t* words = reinterpret_cast<const i32x4_t*>(h + head);
  i32x4_t w[HW];
  auto next_words = [&](int i) {
#pragma unroll
    for (int k = 0; k < HW; ++k)
      if (i + k * NT < whole) w[k] = words[i + k * NT];
  };
  next_words(tid);
  int ends[2] = {-1, -1};               // tokens before and behind the words
  if (counts && tid < head) ends[0] = h[tid];
  if (counts && tid < total - tail) ends[1] = h[tail + tid];
  const int* b = a.bias_tokens + (long)slot * a.biases;
  const int bias0 = biased && tid < a.biases ? b[tid] : -1;
  // in place only what is rewritten is read
  if (!same || masked)
#pragma unroll
    for (int u = 0; u < U; ++u) load(u);
  uint32_t bits[U];
  const int* mask = a.mask + (long)slot * a.words;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i0 = base + (u * NT + tid) * VEC;
    bits[u] = ~0u;
    const int lo = max(i0, 0), hi = min(i0 + VEC, V) - 1;
    if (!masked || lo > hi) continue;
    // bit j: token i0 + j is allowed
    const uint64_t two = (uint32_t)mask[lo >> 5] |
                         (uint64_t)(uint32_t)mask[hi >> 5] << 32;
    bits[u] = (hi >> 5 == lo >> 5 ? (uint32_t)two >> (lo & 31)
                                  : (uint32_t)(two >> (lo & 31))) << (lo - i0);
  }
  const float* values = a.bias_values + (long)slot * a.biases;
  if (counts || biased) {
#pragma unroll
    for (int i = tid * 4; i < CHUNK; i += NT * 4)
      *reinterpret_cast<i32x4_t*>(lds + i) = i32x4_t{0, 0, 0, 0};
    lds_barrier();
    if (counts) {
      auto count = [&](int i, int token) {
        const int t = token - base;
        if ((unsigned)t >= (unsigned)CHUNK || token < 0) return;
        if (i < prompt) atomicOr(&lds[at(t)], SEEN);
        else atomicAdd(&lds[at(t)], 1u);
      };
      count(tid, ends[0]);
      count(tail + tid, ends[1]);
      for (int i = tid; i < whole; i += HW * NT) {
        if (i != tid) next_words(i);
#pragma unroll
        for (int k = 0; k < HW; ++k)
          if (i + k * NT < whole)
#pragma unroll
            for (int j = 0; j < 4; ++j) count(head + (i + k * NT) * 4 + j, w[k][j]);
      }
      lds_barrier();
    }
    // the last entry of a token holds; the lower bits stand still by now
    if (biased) {
      for (int i = tid; i < a.biases; i += NT) {
        const int token = i == tid ? bias0 : b[i], t = token - base;
        if ((unsigned)t < (unsigned)CHUNK && token >= 0)
          atomicMax(&lds[at(t)], (uint32_t)(i + 1) << BIAS |
                                     (lds[at(t)] & ((1u << BIAS) - 1)));
      }
      lds_barrier();
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t0 = (u * NT + tid) * VEC, i0 = base + t0;
    if (i0 >= V) continue;
    if (counts || biased) {
      uint32_t c[VEC], any = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) any |= c[j] = lds[at(t0 + j)];
      if (same && !masked) {
        if (any == 0) continue;
        load(u);
      }
      if (any != 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (c[j] != 0)
            v[u].v[j] = rounded<T>(ruled((float)v[u].v[j], c[j], rep, freq, pres, values));
    }
    if (masked) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (!(bits[u] >> j & 1)) v[u].v[j] = rounded<T>(-INFINITY);
    }
    if (i0 >= 0 && i0 + VEC <= V) {
      *reinterpret_cast<Word*>(to + i0) = v[u];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (i0 + j >= 0 && i0 + j < V) to[i0 + j] = v[u].v[j];
    }
  }
}

// Tokens at the ends of their slots' histories: row i's behind those of the rows
// before it with the same slot.  One block
__global__ __launch_bounds__(256) void append_tokens_kernel(
    int* history, int* total_len, const int* rows, const int64_t* tokens, int N,
    int slots, int cap) {
  for (int step = 0; step < 2; ++step) {
    for (int i = threadIdx.x; i < N; i += 256) {
      const int s = rows[i];
      if (s < 0 || s >= slots) continue;
      int before = 0, behind = 0;
      for (int j = 0; j < N; ++j)
        if (rows[j] == s) j < i ? ++before : j > i ? ++behind : 0;
      const long had = max(total_len[s], 0), at = had + before;
      if (step == 0) {
        const int64_t t = tokens[i];
        if (at < cap) history[(long)s * cap + at] = t >= 0 && t < (1L << 31) ? (int)t : -1;
      } else if (behind == 0 && had < cap) {
        total_len[s] = (int)min(at + 1, (long)cap);
      }
    }
    __syncthreads();
  }
}

static void check_ints(const torch::Tensor& t, const torch::Tensor& by, const char* what) {
  TORCH_CHECK(t.device() == by.device() && t.scalar_type() == torch::kInt32 &&
                  t.is_contiguous(),
              what, ": contiguous int32 on the same device");
}

void adjust_logits(torch::Tensor out, torch::Tensor logits, torch::Tensor rows,
                   torch::Tensor history, torch::Tensor prompt_len,
                   torch::Tensor total_len, torch::Tensor repetition,
                   torch::Tensor frequency, torch::Tensor presence,
                   torch::Tensor bias_tokens, torch::Tensor bias_values,
                   torch::Tensor mask, torch::Tensor masked) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && out.sizes() == logits.sizes() &&
                  out.device() == logits.device() &&
                  out.scalar_type() == logits.scalar_type(),
              "adjust_logits: logits and out (N, V) of one type and device");
  const long N = logits.size(0), V = logits.size(1);
  TORCH_CHECK((V <= 1 || (logits.stride(1) == 1 && out.stride(1) == 1)) &&
                  V < (1L << 30),
              "adjust_logits: rows of adjacent numbers");
  TORCH_CHECK(((out.data_ptr() == logits.data_ptr() && out.strides() == logits.strides()) ||
               !rows_overlap(out, logits)) && (N <= 1 || out.stride(0) >= V),
              "adjust_logits: out is logits or apart from it, its rows from each other");
  for (const auto& t : {rows, history, prompt_len, total_len, bias_tokens, mask, masked})
    check_ints(t, logits, "adjust_logits");
  const long R = history.size(0), cap = history.size(1), nb = bias_tokens.size(1);
  TORCH_CHECK(rows.dim() == 1 && rows.size(0) == N && prompt_len.numel() == R &&
                  total_len.numel() == R && masked.numel() == R && mask.size(0) == R &&
                  mask.size(1) == (V + 31) / 32 && bias_tokens.size(0) == R &&
                  bias_values.sizes() == bias_tokens.sizes(),
              "adjust_logits: rules of another shape");
  for (const auto& t : {repetition, frequency, presence, bias_values})
    TORCH_CHECK(t.device() == logits.device() && t.scalar_type() == torch::kFloat32 &&
                    t.is_contiguous() && (t.dim() == 2 || t.numel() == R),
                "adjust_logits: contiguous fp32 rules");
  TORCH_CHECK(cap <= MOST_TOKENS && nb <= MOST_BIASES, "adjust_logits: at most ",
              MOST_TOKENS, " tokens and ", MOST_BIASES, " biases a slot");
  if (N == 0 || V == 0) return;
  const c10::DeviceGuard guard(logits.device());
  const Rules a{rows.data_ptr<int>(), history.data_ptr<int>(),
                prompt_len.data_ptr<int>(), total_len.data_ptr<int>(),
                repetition.data_ptr<float>(), frequency.data_ptr<float>(),
                presence.data_ptr<float>(), bias_tokens.data_ptr<int>(),
                bias_values.data_ptr<float>(), mask.data_ptr<int>(),
                masked.data_ptr<int>(), (int)R, (int)cap, (int)nb, (int)mask.size(1)};
  auto go = [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = 16 / sizeof(T);
    const uintptr_t apart = (uintptr_t)logits.data_ptr() ^ (uintptr_t)out.data_ptr();
    const bool wide = (apart & 15) == 0 &&
                      ((logits.stride(0) - out.stride(0)) * sizeof(T) & 15) == 0;
    // (a row that starts inside a word has one group more)
    const int chunk = wide ? NT * VEC * 2 : NT * 16;
    const long chunks = (V + (wide ? VEC : 0) + chunk - 1) / chunk;
    TORCH_CHECK(N * chunks < (1L << 31), "adjust_logits: too many rows");
    auto kern = wide ? logit_rules_kernel<T, true, 2> : logit_rules_kernel<T, false, 16>;
    kern<<<dim3((unsigned)(N * chunks)), dim3(NT), 0, at::hip::getCurrentHIPStream()>>>(
        (T*)out.data_ptr(), (const T*)logits.data_ptr(), a, (int)V, logits.stride(0),
        out.stride(0), (int)chunks);
  };
  if (logits.scalar_type() == torch::kBFloat16) go(bf16_t{});
  else if (logits.scalar_type() == torch::kFloat32) go(float{});
  else TORCH_CHECK(false, "adjust_logits: dtype must be bf16 or fp32");
  HIP_CHECK_KERNEL();
  written(out);
}

void append_tokens(torch::Tensor history, torch::Tensor total_len, torch::Tensor rows,
                   torch::Tensor tokens) {
  TORCH_CHECK(history.is_cuda() && history.dim() == 2 && rows.dim() == 1 &&
                  total_len.numel() == history.size(0),
              "append_tokens: history (slots, capacity), rows (N)");
  for (const auto& t : {history, total_len, rows}) check_ints(t, history, "append_tokens");
  TORCH_CHECK(tokens.device() == history.device() && tokens.is_contiguous() &&
                  tokens.scalar_type() == torch::kInt64 && tokens.numel() == rows.numel(),
              "append_tokens: tokens (N) int64");
  TORCH_CHECK(rows.numel() <= 16384, "append_tokens: at most 16384 rows");
  if (rows.numel() == 0) return;
  const c10::DeviceGuard guard(history.device());
  append_tokens_kernel<<<dim3(1), dim3(256), 0, at::hip::getCurrentHIPStream()>>>(
      history.data_ptr<int>(), total_len.data_ptr<int>(), rows.data_ptr<int>(),
      tokens.data_ptr<int64_t>(), (int)rows.numel(), (int)history.size(0),
      (int)history.size(1));
  HIP_CHECK_KERNEL();
}
