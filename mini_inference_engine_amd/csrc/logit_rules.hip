// Rules on a row's logits before a token is chosen from it: penalties for tokens that are already there, biases on single
// tokens, a mask of the tokens that may come.  For token v of a row whose request's text is h_0 .. h_(n-1), of which the first
// p are its prompt, with c the number of v's among h_p .. h_(n-1):
//   z1 = z / repetition if z > 0, else z * repetition,  where v occurs in the text, else z
//   z2 = (z1 - frequency * c) - presence                where c > 0, else z1
//   z3 = z2 + the row's bias of v (the last one listed, where v is listed more than once)
//   z4 = z3 where the row's mask has bit v set (or the row has no mask), else -infinity, whatever z3 is
// every operation rounded by itself in 32 bits.  adjust: z4 itself; choose: what sampling.hip chooses from z4, bit for bit,
// without z4 ever being in memory.
//
// A workgroup has a slice of one row's vocabulary.  It counts its slice's tokens in the LDS (one word a token: occurrences in the
// output, and two bits for "in the text" and "has a bias"), by integer operations, whose order does not matter, then streams
// the slice's logits, asked for before the text is read, past those words.  Every slice reads the row's whole text; it comes from the L2 for
// all slices but one.  Biases are settled after that, the last of a token's entries first.
//
// What bounds it, of what a call cannot do without (MI355X; "the same" is one call's inputs again and again, "others" several calls' in turn): 256 rows
// of 128,256 with texts of 700 to 2,000 tokens chosen in 43 us of the same, 44 to 46 of others, where the 134 MB of logits take 19 at the rate of a
// kernel that only reads.  Reading alone, in this division, takes 25 with the join of the slices, texts 7.5, biases 5, masks 1 and noise on a quarter
// of the rows 6, all of them vector instructions, which keep the units busy for 65 % of the time.  192 rows with texts of 4,000 to 12,000 adjusted in
// 42 us of the same, 47 to 49 of others, where their 205 MB take 40 at the rate of a large copy; results are stored past the L2s, where they would push
// out what the slices share (49 of the same and 50 of others otherwise; logits read that way: 46.5 and, choosing, 44.5 of the same).  Recording a step's
// tokens is a call of 8 us, of 1 token or 2,048: the host's.  Tried and slower (us of the two, where the present form took 52 and 53): slices of 8,192 on 512
// threads (62 and 59) or on 256 (62 and 59), of 6,144 (52.5 and 53); tokens with a word gathered in a list and taken by themselves (64 and 57); a bound
// on the noise by one logarithm before the exact two (63); text and list asked for before the words are cleared (62 and 79).  An entry of the list that
// claims its token before the text is counted saves three barriers and 1 %.
#include "launch.hpp"
#include "sampling.hpp"
#include <type_traits>
#pragma clang fp contract(off)      // the formulas' roundings, one by one

constexpr int THREADS = 256;
constexpr int AHEAD = 4;                               // reads of four logits a thread, all on their way at once
constexpr int ARRIVED = 32;                            // numbers from one row's counter to the next: a cache line each, so that rows do not wait for one another
constexpr int MOST_SLICE = THREADS * 4 * AHEAD, LEAST_SLICE = THREADS * 4;
// four numbers wherever they begin
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
constexpr uint32_t SEEN = 0x80000000u, BIASED = 0x40000000u, TIMES = 0x3FFFFFFFu;

struct Rules {
  const int* history;      // [slots, most] tokens by position, or null: no penalties
  long history_ld;
  int slots, most;
  const int* slot;         // [rows] of history
  const int* length;       // [rows] tokens of the text
  const int* prompt;       // [rows] of these, the prompt's
  const float* repetition; // [rows] each
  const float* presence;
  const float* frequency;
  const int* bias_starts;  // [rows + 1] into the lists, or null: no biases
  const int* bias_tokens;
  const float* bias_values;
  int biases;              // entries of the lists
  const uint32_t* masks;   // [num_masks, mask_ld] bit v % 32 of word v / 32, or null: no masks
  long mask_ld;
  int num_masks;
  const int* mask_row;     // [rows]; what is not an index of a mask: none
};

__device__ __forceinline__ int clamp_int(int x, int low, int high) { return x < low ? low : (x > high ? high : x); }

struct RowRules {
  float repetition, presence, frequency;
};

// penalties
__device__ __forceinline__ float apply_rules(float z, uint32_t w, const RowRules& r) {
  if (w == 0) return z;
  if (w & SEEN) z = z > 0.f ? z / r.repetition : z * r.repetition;
  const uint32_t c = w & TIMES;
  if (c) {
    z = z - r.frequency * (float)c;
    z = z - r.presence;
  }
  return z;
}

__device__ __forceinline__ unsigned long long pack_candidate(float v, int i) {
  return ((unsigned long long)__float_as_uint(v) << 32) | (uint32_t)i;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int from_lane(int x) { return __builtin_amdgcn_update_dpp(x, x, CTRL, ROWS, 0xF, false); }

// The largest (or smallest) of a wave's 64 numbers, for every lane.
template <bool LARGEST>
__device__ __forceinline__ int wave_extreme(int x) {
  auto pick = [](int a, int b) { return LARGEST ? (a > b ? a : b) : (a < b ? a : b); };
  x = pick(x, from_lane<0x111, 0xF>(x));       // from 1, 2, 4 and 8 lanes before in a row of 16, then from the last lane of the row and the half before
  x = pick(x, from_lane<0x112, 0xF>(x));
  x = pick(x, from_lane<0x114, 0xF>(x));
  x = pick(x, from_lane<0x118, 0xF>(x));
  x = pick(x, from_lane<0x142, 0xA>(x));
  x = pick(x, from_lane<0x143, 0xC>(x));
  return __builtin_amdgcn_readlane(x, 63);
}

// The best of a wave's candidates, for every lane: floats (none NaN) in order as integers (-0 as 0), then the lowest index of the largest.
__device__ __forceinline__ void wave_best(float& bv, int& bi) {
  auto turn = [](int bits) { return bits ^ (bits >> 31 & 0x7FFFFFFF); };
  const int mine = turn(__float_as_int(bv + 0.f)), most = wave_extreme<true>(mine);
  bi = wave_extreme<false>(mine == most ? bi : 0x7FFFFFFF);
  bv = __int_as_float(turn(most));
}

// The token of the best of n candidates, for every lane of a wave.
__device__ __forceinline__ int best_of_row(const unsigned long long* best, int n) {
  float bv = -INFINITY;
  int bi = 0x7FFFFFFF;
  for (int i = threadIdx.x; i < n; i += 64) {
    const unsigned long long c = __hip_atomic_load(&best[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sample_better(__uint_as_float((uint32_t)(c >> 32)), (int)(uint32_t)c, bv, bi);
  }
  wave_best(bv, bi);
  return bi == 0x7FFFFFFF ? 0 : bi;
}

// Grid (slices of a row, rows), a workgroup each.  CHOOSE: its best candidate to best [rows, workgroups], or,
// of a row that has one workgroup, the token to ``chosen``; else the adjusted logits to ``out``.  With ``arrived`` (a counter a
// row, 0 before and after) the last workgroup of a row to arrive joins the row's candidates: one launch instead of two.
template <bool CHOOSE>
__global__ void __launch_bounds__(THREADS, 8)
rules_kernel(const float* logits, long ld, Rules rules, int V, int slice, float* out, long out_ld,
             const float* __restrict__ temperatures, const long long* __restrict__ seeds, const int* __restrict__ counters,
             unsigned long long* best, int* arrived, int* __restrict__ chosen) {
  extern __shared__ __align__(16) uint32_t words[];                   // [slice]
  __shared__ float wave_v[THREADS / 64];
  __shared__ int wave_i[THREADS / 64];
  const int r = blockIdx.y, tid = threadIdx.x;

  // Everything a row says of itself is asked for at once, from the logits where a rule is absent (what is read there is not used): one wait
  // and not one behind each test.
  auto of_row = [&](const auto* p, int i) {
    using N = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
    return *(p ? p + i : reinterpret_cast<const N*>(logits));
  };
  RowRules row{of_row(rules.repetition, r), of_row(rules.presence, r), of_row(rules.frequency, r)};
  const int in_slot = of_row(rules.slot, r), in_length = of_row(rules.length, r), in_prompt = of_row(rules.prompt, r);
  const int bias_a = of_row(rules.bias_starts, r), bias_b = of_row(rules.bias_starts, r + 1), in_mask = of_row(rules.mask_row, r);
  float temperature = 0.f;
  uint32_t key = 0;
  if (CHOOSE) {
    temperature = temperatures[r];
    key = sample_key((unsigned long long)seeds[r], counters[r]);
  }
  const bool penalised = rules.history && (row.repetition != 1.f || row.presence != 0.f || row.frequency != 0.f) && in_slot >= 0 && in_slot < rules.slots;
  const int* text = penalised ? rules.history + (size_t)in_slot * rules.history_ld : nullptr;
  const int length = penalised ? clamp_int(in_length, 0, rules.most) : 0, prompt = clamp_int(in_prompt, 0, length);
  const int first_bias = rules.bias_starts ? clamp_int(bias_a, 0, rules.biases) : 0;
  const int listed = rules.bias_starts ? clamp_int(bias_b, first_bias, rules.biases) - first_bias : 0;
  const int* list = rules.bias_tokens + first_bias;
  const float* list_values = rules.bias_values + first_bias;
  const uint32_t* mask = rules.masks && in_mask >= 0 && in_mask < rules.num_masks ? rules.masks + (size_t)in_mask * rules.mask_ld : nullptr;
  const bool noisy = CHOOSE && temperature > 0.f;
  const float inv_t = noisy ? 1.0f / temperature : 1.f;
  float bv = -INFINITY;
  int bi = 0x7FFFFFFF;
  const bool counted = length > 0 || listed > 0;                      // (the same in the whole workgroup)
  const int begin = blockIdx.x * slice;
  const int n = min(slice, V - begin), n4 = n & ~3;
  const float* z0 = logits + (size_t)r * ld + begin;
  // The list's first entries, one a thread, then the slice's logits and mask are asked for before the text is read.
  const unsigned own = tid < listed ? (unsigned)list[tid] - (unsigned)begin : ~0u;
  const float own_value = tid < listed ? list_values[tid] : 0.f;
  f32x4_any z[AHEAD];
  uint32_t bits[AHEAD];
#pragma unroll
  for (int k = AHEAD - 1; k >= 0; --k) {
    const int i = (k * THREADS + tid) * 4;
    if (i < n4) {
      z[k] = *reinterpret_cast<const f32x4_any*>(z0 + i);
      bits[k] = mask ? mask[(begin + i) >> 5] >> ((begin + i) & 31) : 15u;
    }
  }
  if (counted) {
    const int zeros = (n + 3) / 4;
    for (int i = tid; i < zeros; i += THREADS) {
      reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    auto count = [&](int token, int i) {
      const unsigned at = (unsigned)token - (unsigned)begin;        // what is no token of the vocabulary is in no slice
      if (at < (unsigned)n) {
        atomicOr(&words[at], SEEN);
        if (i >= prompt) atomicAdd(&words[at], 1u);
      }
    };
    const int length4 = length & ~3;
    constexpr int READS = 4;                                        // on their way together
    for (int i0 = tid * 4; i0 < length4; i0 += READS * THREADS * 4) {
      i32x4_any t[READS];
#pragma unroll
      for (int k = 0; k < READS; ++k) {
        const int i = i0 + k * THREADS * 4;
        t[k] = *reinterpret_cast<const i32x4_any*>(text + (i < length4 ? i : i0));
      }
#pragma unroll
      for (int k = 0; k < READS; ++k) {
        const int i = i0 + k * THREADS * 4;
        if (i >= length4) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) count(t[k][j], i + j);
      }
    }
    if (length4 + tid < length) count(text[length4 + tid], length4 + tid);
    if (own < (unsigned)n) atomicOr(&words[own], BIASED);
    for (int i = tid + THREADS; i < listed; i += THREADS) {
      const unsigned at = (unsigned)list[i] - (unsigned)begin;
      if (at < (unsigned)n) atomicOr(&words[at], BIASED);
    }
    __syncthreads();
  }
  float* o0 = CHOOSE ? nullptr : out + (size_t)r * out_ld + begin;
  // A thread goes through its tokens from the last to the first, so that one comparison keeps the first of equals (and no NaN).
  auto keep = [&](float y, int i) {
    const float v = sample_value(y, begin + i, noisy, inv_t, key);
    const bool better = v >= bv;
    bv = better ? v : bv;
    bi = better ? begin + i : bi;
  };
  if (n4 + tid < n) {                                               // up to three at the end of the row
    const int i = n4 + tid;
    const uint32_t w = counted ? words[i] : 0;
    const bool may = !mask || (mask[(begin + i) >> 5] >> ((begin + i) & 31) & 1);
    const float z1 = z0[i], y = w & BIASED ? z1 : may ? apply_rules(z1, w, row) : -INFINITY;
    if (!CHOOSE) o0[i] = y;
    else if (!(w & BIASED)) keep(y, i);
  }
#pragma unroll
  for (int k = AHEAD - 1; k >= 0; --k) {
    const int i = (k * THREADS + tid) * 4;
    if (i >= n4) continue;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (counted) w = *reinterpret_cast<const uint4*>(words + i);
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const uint32_t wj = j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w;
      const float y = bits[k] >> j & 1 ? apply_rules(z[k][j], wj, row) : -INFINITY;
      if (wj & BIASED) continue;                                    // left as it is to the list, below
      if (CHOOSE) keep(y, i + j);
      else z[k][j] = y;
    }
    if (!CHOOSE) __builtin_nontemporal_store(z[k], reinterpret_cast<f32x4_any*>(o0 + i));
  }
  // The tokens with a bias, a thread an entry of the list, the list's end first.  Of several entries of a token the last one
  // has it: within a round the largest thread that asks for it, and what a round has settled has lost its mark for those before.
  for (int i0 = (listed - 1) / THREADS * THREADS; listed > 0 && i0 >= 0; i0 -= THREADS) {
    const int e = i0 + tid;
    const unsigned at = i0 == 0 ? own : e < listed ? (unsigned)list[e] - (unsigned)begin : ~0u;
    const bool mine = at < (unsigned)n;
    if (!CHOOSE) MIE_VMCNT(0);                                      // the logits as they were are in memory
    __syncthreads();
    const uint32_t w = mine ? words[at] : 0;
    const bool asks = w & BIASED;
    __syncthreads();
    if (asks) words[at] = 0;
    __syncthreads();
    if (asks) atomicMax(&words[at], (uint32_t)tid + 1);
    __syncthreads();
    if (asks && words[at] == (uint32_t)tid + 1) {
      const int v = begin + (int)at;
      const bool may = !mask || (mask[v >> 5] >> (v & 31) & 1);
      const float y = may ? apply_rules(z0[at], w & ~BIASED, row) + (i0 == 0 ? own_value : list_values[e]) : -INFINITY;
      if (CHOOSE) sample_consider(y, v, noisy, inv_t, key, bv, bi);
      else o0[at] = y;
    }
  }
  if (!CHOOSE) return;
  wave_best(bv, bi);
  if ((tid & 63) == 0) { wave_v[tid >> 6] = bv; wave_i[tid >> 6] = bi; }
  __syncthreads();
  if (tid >= 64) return;
  int last = 0;
  if (tid == 0) {
    for (int i = 1; i < THREADS / 64; ++i) sample_better(wave_v[i], wave_i[i], bv, bi);
    if (gridDim.x == 1) {
      chosen[r] = bi == 0x7FFFFFFF ? 0 : bi;
    } else {
      // Past the L2s, which workgroups on different dies do not share, by itself: a release of the whole L2 costs far more.
      __hip_atomic_store(&best[(size_t)r * gridDim.x + blockIdx.x], pack_candidate(bv, bi), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (arrived) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // it is there before the row's counter says so
        last = __hip_atomic_fetch_add(&arrived[(size_t)r * ARRIVED], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
      }
    }
  }
  if (!__shfl(last, 0, 64)) return;
  asm volatile("" ::: "memory");
  const int token = best_of_row(best + (size_t)r * gridDim.x, gridDim.x);
  if (tid == 0) {
    chosen[r] = token;
    __hip_atomic_store(&arrived[(size_t)r * ARRIVED], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// The best of a row's slices, one wave a row.
__global__ void __launch_bounds__(64)
best_of_slices_kernel(const unsigned long long* best, int* __restrict__ chosen, int slices) {
  const int token = best_of_row(best + (size_t)blockIdx.x * slices, slices);
  if (threadIdx.x == 0) chosen[blockIdx.x] = token;
}

// history[slot of the token's row, its position] = the token, of every token of a step.
__global__ void __launch_bounds__(256)
record_tokens_kernel(int* __restrict__ history, long ld, int slots, int most, const int* __restrict__ ids, const int* __restrict__ taken_from,
                     const int* __restrict__ earlier, int num_earlier, const int* __restrict__ token_row, const int* __restrict__ state_slots,
                     int rows, const int* __restrict__ positions, int T) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int r = token_row[t], p = positions[t], from = taken_from ? taken_from[t] : -1;
  if (r < 0 || r >= rows || p < 0 || p >= most) return;
  const int s = state_slots[r];
  if (s < 0 || s >= slots) return;
  history[(size_t)s * ld + p] = from >= 0 && from < num_earlier ? earlier[from] : ids[t];
}

MIE_EXPORT const char* logit_rules_last_error() { return g_mie_error; }

// Tokens a workgroup takes: fewer as long as the workgroups are few.  (Kernels alone, us, choosing and adjusting: 8 rows of 8,000 6.5 and 4.2, 9.8 and 6.1
// a row in one workgroup of 1,024 threads, 256 rows of 5,000 9.1 and 6.6 where those take 8.4 and 6.1.)  Four a compute unit are enough, at eight every text is read too
// often (32 rows of 128,256 12.0, 15.8), at two the units are not filled (64 rows of 32,000 9.5, 10.9).
static int slice_for(int rows, int V) {
  int slice = MOST_SLICE;
  while (slice > LEAST_SLICE && (long)rows * ((V + slice - 1) / slice) < 4L * mie_compute_units()) slice /= 2;
  return slice;
}

// Workgroups a row.
MIE_EXPORT int mie_rules_slices(int rows, int V) {
  const int slice = slice_for(rows, V);
  return (V + slice - 1) / slice;
}

static int check_rules(const char* what, const Rules& r, int rows, int V, long ld) {
  if (V <= 0 || V > 1 << 30 || ld < V) MIE_FAIL("%s: vocabulary %d, leading dim %ld", what, V, ld);
  if (rows > 65535) MIE_FAIL("%s: %d rows, at most 65535", what, rows);
  if (r.history && (r.most < 0 || r.history_ld < r.most || r.slots < 0)) MIE_FAIL("%s: history of %d slots, %d positions, %ld apart", what, r.slots, r.most, r.history_ld);
  if (r.masks && (r.mask_ld < (V + 31) / 32 || r.num_masks < 0)) MIE_FAIL("%s: masks of %ld words for a vocabulary of %d", what, r.mask_ld, V);
  return 0;
}

template <bool CHOOSE>
static int launch_rules(const char* what, const float* logits, long ld, const Rules& rules, int rows, int V, float* out, long out_ld,
                        const float* temperatures, const long long* seeds, const int* counters, unsigned long long* best, int* arrived,
                        int* chosen, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (check_rules(what, rules, rows, V, ld)) return -1;
  const int slice = slice_for(rows, V), slices = (V + slice - 1) / slice;
  hipLaunchKernelGGL(rules_kernel<CHOOSE>, dim3(slices, rows), dim3(THREADS), slice * 4, stream, logits, ld, rules, V, slice, out, out_ld, temperatures,
                     seeds, counters, best, arrived, chosen);
  MIE_CHECK_LAUNCH(what);
  if (CHOOSE && slices > 1 && !arrived) {
    hipLaunchKernelGGL(best_of_slices_kernel, dim3(rows), dim3(64), 0, stream, best, chosen, slices);
    MIE_CHECK_LAUNCH(what);
  }
  return 0;
}

#define RULE_ARGS                                                                                                                    \
  const int *history, long history_ld, int slots, int most, const int *slot, const int *length, const int *prompt,                    \
      const float *repetition, const float *presence, const float *frequency, const int *bias_starts, const int *bias_tokens,         \
      const float *bias_values, int biases, const uint32_t *masks, long mask_ld, int num_masks, const int *mask_row
#define RULES                                                                                                                         \
  Rules { history, history_ld, slots, most, slot, length, prompt, repetition, presence, frequency, bias_starts, bias_tokens,          \
          bias_values, biases, masks, mask_ld, num_masks, mask_row }

MIE_EXPORT int mie_adjust_logits(const float* logits, long ld, RULE_ARGS, float* out, long out_ld, int rows, int V, hipStream_t stream) {
  if (rows > 0 && out_ld < V) MIE_FAIL("adjust_logits: rows of the result %ld apart for a vocabulary of %d", out_ld, V);
  return launch_rules<false>("adjust_logits", logits, ld, RULES, rows, V, out, out_ld, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, stream);
}

// best: [rows, mie_rules_slices] and, unless null (a second launch then joins the slices), arrived: [32 rows], zero; both unused where there is one slice,
// and nobody else's while the call runs.
MIE_EXPORT int mie_choose_by_rules(const float* logits, long ld, RULE_ARGS, const float* temperatures, const long long* seeds,
                                   const int* counters, unsigned long long* best, int* arrived, int* chosen, int rows, int V,
                                   hipStream_t stream) {
  return launch_rules<true>("sample", logits, ld, RULES, rows, V, nullptr, 0, temperatures, seeds, counters, best, arrived, chosen, stream);
}

MIE_EXPORT int mie_record_tokens(int* history, long ld, int slots, int most, const int* ids, const int* taken_from, const int* earlier,
                                 int num_earlier, const int* token_row, const int* state_slots, int rows, const int* positions, int T,
                                 hipStream_t stream) {
  if (T <= 0) return 0;
  if (ld < most) MIE_FAIL("record_tokens: history of %d positions, %ld apart", most, ld);
  hipLaunchKernelGGL(record_tokens_kernel, dim3((T + 255) / 256), dim3(256), 0, stream, history, ld, slots, most, ids, taken_from, earlier,
                     num_earlier, token_row, state_slots, rows, positions, T);
  MIE_CHECK_LAUNCH("record_tokens");
  return 0;
}
