// Attention of single-token rows whose requests share the first part of their cache, the shared keys read once for all of them.
// Caches: keys [pages, Hkv, page, D], values [pages, Hkv, D, page], bfloat16 or float32.
//
// softmax(s q . k) v splits over any cut of the keys: with m a running maximum, l = sum exp2(x - m) and o = sum exp2(x - m) v of
// each part, parts join by their log-sum-exps m + log2 l.  A plan made on the host (kernels/shared_prefix.py) cuts a step into
// items: columns x keys of one kv head.  A column is one query head of one row; the columns of an item over shared keys are the
// group's query heads of up to 64 CT / G rows (G query heads a kv head), those of an item over a row's own keys are its G query heads.
// One workgroup of four waves an item and kv head.  With v_mfma_f32_16x16x32_bf16 (float32: 16x16x4)
//   S^T[key, column]  = K[key, d] . Q^T[d, column]        A = 16 keys, B = 16 columns
//   O^T[dim, column] += V^T[dim, key] . P^T[key, column]
// The scores come out with lane % 16 = column and 4 consecutive rows a lane group.  In bfloat16 the 32 keys are dealt to the two score
// tiles' rows so that lane group g ends up with keys 8 g .. 8 g + 7, which is what the second product takes of both operands; in float32 every
// one of the second product's steps of 4 keys takes one number of each lane group.  Probabilities never leave registers; they are rounded to
// bfloat16 for the second product as the operand of its kind, their sum is of what they were before.
//
// Keys and values come into the LDS by loads that write it directly, and the waves share the work out in one of two ways:
//   more than 16 columns: all waves bring in a stage (64 keys, 32 where a key has more than 256 bytes), each takes 16 CT of the columns through it
//   up to 16 columns: each wave brings in and takes every fourth 32 keys, and the waves join in the LDS at the end; with the first way one
//   wave would compute and three wait (a row's 1,024 keys of 128 numbers 19.5 us, 12.8 this way, of 4,096 63.7 and 40.9).  Of keys of more than 256
//   bytes two waves take every second 32: their LDS then leaves room for a second workgroup (150 rows of 16 / 2 heads of 256 with up to 308 keys
//   25.4 -> 16.7 us).  Where such items are many and short, each of these waves has one to itself, and nothing is joined in the LDS.
//
// What bounds it (MI355X).  256 rows of 32 / 8 heads of 128 behind 8,192 shared keys with 1 to 1,024 of their own, 106 to 111 us with the join.  In the same
// run the 540 MB of own keys alone take 88 to 92 (5.9 TB/s), the 34 GFLOP over shared keys alone 63 to 66, for the most part hidden behind them as long as
// the own keys' waves, which wait for no other wave, share the units (with four waves a row 131 to 141).  Many columns alone are a chain of LDS reads, products and
// softmax: of 1,024 keys of 128 a workgroup of 128 columns takes 34 us by itself, two on a unit 51.  8 rows behind 30,000 keys 32.5 us for 134 MB (4.1
// TB/s).  32 rows behind 2,000 keys 18 to 19 us, 4 of them the join: a workgroup's first loads, last stores and one stage take 7 us.
#include "attention_bf16_common.hpp"
#include "launch.hpp"
#include <type_traits>

constexpr int WAVES = 4;
// Tiles of 16 columns a wave: two in bfloat16, as far as their outputs have room in the registers.  (In float32 the matrix instructions bound what
// many columns cost, and two workgroups on a compute unit do more than one of twice the columns.)
constexpr int MOST_TILES = D <= 128 ? 2 : 1;

// 16 bytes a lane from a lane's own address into the LDS at byte `at` + 16 lane (waits are the kernel's own)
__device__ __forceinline__ void lane_load_to_lds(const char* from, uint32_t at) {
  uint32_t written;
  asm volatile(
    "s_mov_b32 m0, %1\n\t"
    "s_nop 0\n\t"
    "global_load_lds_dwordx4 %2, off"
    : "={m0}"(written)
    : "s"(at), "v"(from)
    : "memory");
}

struct SharedItem {
  int first_row;      // whose block table finds the keys
  int columns;        // of the item's rows: rows x G
  int col0;           // first of them that the item takes
  int key_begin, key_end;
  int part;           // which of its rows' partial results
  int unused[2];
};

template <typename T, int CT>
struct Layout {
  static constexpr int ES = sizeof(T);
  static constexpr int ROW = D * ES;                        // bytes of a key
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int TURN = CHUNKS % 8 == 0 ? 7 : CHUNKS % 4 == 0 ? 3 : 1;
  static constexpr int VROW = 16 * ES;                      // bytes of 16 keys' values of one dim
  static constexpr int TILE = BLOCK_KEYS * ROW;             // keys of 32; their values take as much
  static constexpr int UNITS = 2 * TILE / 1024;             // loads of 1 KB that bring both
  static constexpr int EACH = (UNITS + WAVES - 1) / WAVES;  // a wave's
  static constexpr bool WHOLE = TILE % 2048 == 0;           // no unit lies across the two halves of 16 keys
  // A stage: what is waited for and computed at once, two times 32 keys where the LDS has room for it (half the barriers, and twice the
  // independent work behind each).
  static constexpr int H = ROW <= 256 ? 2 : 1;
  static constexpr int KEYS = H * BLOCK_KEYS;
  static constexpr int STAGE = H * 2 * TILE;
  static constexpr int STAGES = STAGE <= 8192 ? 6 : STAGE <= 16384 ? 4 : 2;
  // Items of up to 16 columns: each wave takes every fourth 32 keys, by itself, in slots of its own.
  static constexpr bool APART = WHOLE;
  static constexpr int SLOT = 2 * TILE;
  static constexpr int SHARERS = ROW <= 256 ? WAVES : 2;    // of the waves: two such workgroups have room on a compute unit
  static constexpr int SLOTS = STAGES * STAGE / (SHARERS * SLOT) > 1 ? 2 : 1;
  static constexpr int JOIN = SHARERS * 16 * (D + 1) * 4;     // the waves' sums, where the slots were
  static constexpr int LDS = !APART ? STAGES * STAGE : STAGES * STAGE > SHARERS * SLOTS * SLOT ? (STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN)
                                                                                             : (SHARERS * SLOTS * SLOT > JOIN ? SHARERS * SLOTS * SLOT : JOIN);
  // 16-byte places are turned by what tells the rows apart that are read at once, so that they lie in different banks
  static __device__ __forceinline__ int key_turn(int r) { return (ES == 2 ? (r & 3) | ((r >> 3 & 1) << 2) : r & 7) & TURN; }
  static __device__ __forceinline__ int value_turn(int d) { return ES == 2 ? d >> 2 & 1 : d >> 1 & 3; }
};

template <typename T, int CT>
__global__ void __launch_bounds__(WAVES * 64, D * sizeof(T) <= (CT == 1 ? 512 : 256) ? 2 : 1)
shared_attention_kernel(const T* __restrict__ q, long q_stride, int q_vec, const T* __restrict__ k_cache, const T* __restrict__ v_cache,
                        T* __restrict__ out, float* __restrict__ o_part, float* __restrict__ lse_part, const int* __restrict__ tables,
                        int max_blocks, int pages, const int* __restrict__ positions, const SharedItem* __restrict__ items, int num_items, int whole_items,
                        const int* __restrict__ row_parts, int Hq, int Hkv, int page, float scale_log2, float sink_log2,
                        const float* __restrict__ head_sinks) {
  using L = Layout<T, CT>;
  constexpr bool HALF = sizeof(T) == 2;
  constexpr int QS = HALF ? KS : D / 16;                    // 16-byte pieces of a column's query that a lane holds
  extern __shared__ __align__(1024) char lds[];
  const int group = blockIdx.x / Hkv, kvh = blockIdx.x - group * Hkv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool solo = L::APART && group >= whole_items;       // every wave has an item of its own
  const int item = solo ? whole_items + (group - whole_items) * L::SHARERS + wave : group;
  if (item >= num_items || (solo && wave >= L::SHARERS)) return;
  const int first_row = items[item].first_row, columns = items[item].columns, col0 = items[item].col0;
  const int key_begin = items[item].key_begin, part = items[item].part;
  int key_end = items[item].key_end;
  const int G = Hq / Hkv;
  const int col = lane & 15, kb = lane >> 4;
  // Keys that no other workgroup reads are loaded with the hint that nobody reads them again: they then push neither the shared keys nor
  // anything else out of the caches (256 rows behind 8,192 keys 177 -> 150 us, their own 1 to 1,024 keys alone 157 -> 97, 8 rows behind
  // 30,000 keys 58 -> 35).
  const bool once = columns <= WAVES * 16 * CT;
  if (columns <= G) {                                       // one row: nothing behind its own key
    const int seen = positions[first_row] + 1;
    key_end = seen < key_end ? seen : key_end;
  }

  const bool apart = L::APART && columns <= 16;             // the waves share out keys, or items, not columns

  // ---- the loads: unit u of 32 keys is 1 KB of their keys or values, a wave takes units wave, wave + 4, ..
  uint32_t rel[L::EACH];
  bool upper[L::EACH], is_key[L::EACH];
#pragma unroll
  for (int i = 0; i < L::EACH; ++i) {
    int u = wave + WAVES * i;
    u = u < L::UNITS ? u : L::UNITS - 1;                    // (a wave without a unit of its own repeats the last one)
    int x = u * 1024 + lane * 16;
    is_key[i] = L::UNITS % (2 * WAVES) == 0 ? i < L::EACH / 2 : u < L::UNITS / 2;
    if (is_key[i]) {
      const int r = x / L::ROW, place = (x - r * L::ROW) / 16;
      upper[i] = L::UNITS % (4 * WAVES) == 0 ? i >= L::EACH / 4 : L::WHOLE ? u >= L::UNITS / 4 : r >= 16;
      rel[i] = (r & 15) * L::ROW + (place ^ L::key_turn(r)) * 16;
    } else {
      x -= L::TILE;
      const int half = x / (D * L::VROW);
      x -= half * D * L::VROW;
      const int d = x / L::VROW, place = (x - d * L::VROW) / 16;
      upper[i] = L::UNITS % (4 * WAVES) == 0 ? i >= 3 * L::EACH / 4 : L::WHOLE ? u >= 3 * (L::UNITS / 4) : half;
      rel[i] = d * page * L::ES + (place ^ L::value_turn(d)) * 16;
    }
  }
  const auto* table = (const __attribute__((address_space(4))) int*)(uintptr_t)(tables + (size_t)first_row * max_blocks);
  // Where a block's keys lie: its halves of 16 keys are in one page each.  Followed from block to block by additions.
  const int blk0 = key_begin & ~(BLOCK_KEYS - 1);       // 32 and not a stage: a cut lies on any 32 keys
  const uint64_t page_bytes = (uint64_t)(uint32_t)Hkv * page * L::ROW;       // of keys; of values as well
  const char* const keys0 = reinterpret_cast<const char*>(k_cache) + (size_t)kvh * page * L::ROW;
  const char* const vals0 = reinterpret_cast<const char*>(v_cache) + (size_t)kvh * page * L::ROW;
  const bool deal = apart && !solo;
  const int stride = deal ? L::SHARERS * BLOCK_KEYS : BLOCK_KEYS, blk1 = blk0 + (deal ? wave * BLOCK_KEYS : 0);
  const int more_pages = stride / page, more_off = stride % page;
  int index[2], off[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    index[t] = (blk1 + 16 * t) / page;
    off[t] = blk1 + 16 * t - index[t] * page;
  }
  struct Places { int pg[2], off[2]; };
  auto find = [&]() {                                       // of the next block of the wave's
    Places p;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      p.pg[t] = table[index[t] < max_blocks ? index[t] : max_blocks - 1];
      p.off[t] = off[t];
      off[t] += more_off;
      const int turn = off[t] >= page ? 1 : 0;
      off[t] -= turn * page;
      index[t] += more_pages + turn;
    }
    return p;
  };
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
  auto issue = [&](uint32_t to, const Places& p) {
    const char *k[2], *v[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t pg = (uint32_t)p.pg[t] < (uint32_t)pages ? p.pg[t] : 0;
      const uint64_t at = pg * page_bytes;
      k[t] = keys0 + at + p.off[t] * L::ROW;
      v[t] = vals0 + at + p.off[t] * L::ES;
    }
#pragma unroll
    for (int i = 0; i < L::EACH; ++i) {
      int u = wave + WAVES * i;
      u = u < L::UNITS ? u : L::UNITS - 1;
      const char* base = is_key[i] ? (upper[i] ? k[1] : k[0]) : (upper[i] ? v[1] : v[0]);
      if constexpr (L::WHOLE) {
        if (once) mie_load_to_lds_nt(base, rel[i], to + u * 1024);
        else mie_load_to_lds(base, rel[i], to + u * 1024);
      }
      else lane_load_to_lds(base + rel[i], to + u * 1024);
    }
  };
  const int blocks = key_end > key_begin ? (key_end - blk0 + BLOCK_KEYS - 1) / BLOCK_KEYS : 0, count = (blocks + L::H - 1) / L::H;
  Places next[L::H];
  // A stage's last 32 keys may lie beyond the item's: they are not asked for, and what the LDS holds in their place is masked.
  auto issue_stage = [&](int n, int stage) {
#pragma unroll
    for (int h = 0; h < L::H; ++h)
      if (h == 0 || n * L::H + h < blocks) issue(lds0 + stage * L::STAGE + h * 2 * L::TILE, next[h]);
  };
  auto find_stage = [&]() {                                 // pages are looked up a stage before their loads
#pragma unroll
    for (int h = 0; h < L::H; ++h) next[h] = find();
  };
  // a wave's own 32 keys: units of one half of 16 keys, and of values, differ by their place alone
  constexpr int KL = L::APART ? L::UNITS / 4 : 1;
  uint32_t koff[KL], voff = 0;
  auto issue_own = [&](int slot, const Places& p) {
    const uint32_t to = lds0 + (wave * L::SLOTS + slot) * L::SLOT;
    const uint32_t half_bytes = L::TILE / 2, dims = 1024 / L::VROW;      // of a unit of values
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint64_t at = ((uint32_t)p.pg[t] < (uint32_t)pages ? (uint32_t)p.pg[t] : 0u) * page_bytes;
      const char* k = keys0 + at + p.off[t] * L::ROW;
#pragma unroll
      for (int j = 0; j < KL; ++j) mie_load_to_lds_nt(k, koff[j], to + t * half_bytes + j * 1024);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint64_t at = ((uint32_t)p.pg[t] < (uint32_t)pages ? (uint32_t)p.pg[t] : 0u) * page_bytes;
      const char* v = vals0 + at + p.off[t] * L::ES;
#pragma unroll
      for (int j = 0; j < KL; ++j) mie_load_to_lds_nt(v + (size_t)(j * dims) * page * L::ES, voff, to + L::TILE + t * half_bytes + j * 1024);
    }
  };
  const int mine = solo ? blocks : wave < L::SHARERS ? (blocks - wave + L::SHARERS - 1) / L::SHARERS : 0;      // of an item of up to 16 columns, 32 keys each
  Places next_own;
  if (apart) {
    if constexpr (L::APART) {
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        const int x = j * 1024 + lane * 16, r = x / L::ROW, place = (x - r * L::ROW) / 16;
        koff[j] = r * L::ROW + (place ^ L::key_turn(r)) * 16;
      }
      const int d = lane * 16 / L::VROW, place = lane * 16 % L::VROW / 16;
      voff = d * page * L::ES + (place ^ L::value_turn(d)) * 16;
      Places first[L::SLOTS];
#pragma unroll
      for (int i = 0; i < L::SLOTS; ++i) first[i] = find();
      next_own = find();
#pragma unroll
      for (int i = 0; i < L::SLOTS; ++i)
        if (i < mine) issue_own(i, first[i]);
    }
  } else {
    find_stage();
#pragma unroll
    for (int i = 0; i < L::STAGES - 1; ++i)
      if (i < count) {
        issue_stage(i, i);
        find_stage();
      }
  }

  // ---- the wave's columns
  int limit[CT];                                            // keys that the lane's column sees end here
  int least = key_end, most = key_begin, tiles = 0;
  Frag qf[CT][QS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c0 = col0 + ((apart ? 0 : wave * CT) + ct) * 16, c = c0 + col;
    const bool ok = c < columns;
    if (c0 < columns) tiles = ct + 1;
    const int r = first_row + (ok ? c / G : 0), head = kvh * G + (ok ? c % G : 0);
    const int seen = positions[r] + 1;
    limit[ct] = ok && seen < key_end ? seen : key_end;
    least = limit[ct] < least ? limit[ct] : least;
    if (ok) most = limit[ct] > most ? limit[ct] : most;
    const T* qp = q + (size_t)r * q_stride + (size_t)head * D;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int d0 = HALF ? s * 32 + kb * 8 : s * 16 + kb * 4;
      qf[ct][s].q = make_uint4(0, 0, 0, 0);
      if (ok && d0 < D) {
        if (q_vec) {
          qf[ct][s].q = *reinterpret_cast<const uint4*>(qp + d0);
        } else {
          T e[16 / sizeof(T)];
#pragma unroll
          for (int j = 0; j < (int)(16 / sizeof(T)); ++j) e[j] = qp[d0 + j];
          __builtin_memcpy(&qf[ct][s].q, e, 16);
        }
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const int a = __shfl_xor(least, o, 64), b = __shfl_xor(most, o, 64);
    least = a < least ? a : least;
    most = b > most ? b : most;
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);

  float m[CT], l[CT];
  f32x4 O[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) O[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // key of a lane's j-th score of the h-th 32 keys
  auto key_at = [&](int blk, int h, int j) {
    return blk + BLOCK_KEYS * h + (HALF ? 8 * kb + j : 16 * (j >> 2) + 4 * kb + (j & 3));
  };

  // a lane's piece s of the keys' rows of score tile t, piece f of the values, of 32 keys in the LDS
  auto key_frag = [&](const char* at, int t, int s) {
    const int r = HALF ? 8 * (col >> 2) + 4 * t + (col & 3) : 16 * t + col;
    const bool beyond = HALF && D % 32 != 0 && s == KS - 1 && kb >= 2;          // the last step of 32 dims is half empty
    Frag a;
    a.q = *reinterpret_cast<const uint4*>(at + r * L::ROW + ((beyond ? 0 : 4 * s + kb) ^ L::key_turn(r)) * 16);
    if (beyond) a.q = make_uint4(0, 0, 0, 0);
    return a;
  };
  auto value_frag = [&](const char* at, int f) {
    const int d = (HALF ? f : f >> 1) * 16 + col, half = HALF ? kb >> 1 : f & 1, place = HALF ? kb & 1 : kb;
    Frag a;
    a.q = *reinterpret_cast<const uint4*>(at + L::TILE + (half * D + d) * L::VROW + (place ^ L::value_turn(d)) * 16);
    return a;
  };
  // 0 * (whatever is in slots that no column sees) must not reach a sum
  auto clear_hidden = [&](Frag& v, int f, int blk, int h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (HALF) {
        const int key = key_at(blk, h, 2 * j);
        v.w[j] &= (key >= key_begin && key < most ? 0x0000FFFFu : 0u) | (key + 1 >= key_begin && key + 1 < most ? 0xFFFF0000u : 0u);
      } else {
        const int key = key_at(blk, h, 4 * (f & 1) + j);
        if (key < key_begin || key >= most) v.w[j] = 0;
      }
    }
  };
  // The first tile of columns through 32 keys whose pieces are in registers.
  auto attend_one = [&](Frag (&a)[2][QS], Frag (&va)[HALF ? DT : 2 * DT], int blk) {
    f32x4 S[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (HALF) {
          S[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][s].v, qf[0][s].v, S[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[t][s].w[j]), __uint_as_float(qf[0][s].w[j]), S[t], 0, 0, 0);
        }
      }
    if (blk < key_begin || blk + BLOCK_KEYS > least) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key_at(blk, 0, j);
        if (key < key_begin || key >= limit[0]) S[j >> 2][j & 3] = -INFINITY;
      }
#pragma unroll
      for (int f = 0; f < (HALF ? DT : 2 * DT); ++f) clear_hidden(va[f], f, blk, 0);
    }
    float mx = S[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, S[j >> 2][j & 3]);
    mx = quad_max(mx) * scale_log2;
    if (__any(mx > m[0] + 8.f)) {
      const float m_new = fmaxf(m[0], mx);
      const float alpha = m[0] == -INFINITY ? 0.f : fast_exp2(m[0] - m_new);
      m[0] = m_new;
      l[0] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) O[0][dt] *= alpha;
    }
    const float base = m[0] == -INFINITY ? 0.f : m[0];
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = fast_exp2(fmaf(S[j >> 2][j & 3], scale_log2, -base));
      l[0] += p[j];
    }
    if constexpr (HALF) {
      Frag pb;
#pragma unroll
      for (int j = 0; j < 4; ++j) pb.w[j] = pack_bf16(p[2 * j], p[2 * j + 1]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) O[0][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[dt].v, pb.v, O[0][dt], 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          O[0][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va[2 * dt + (j >> 2)].w[j & 3]), p[j], O[0][dt], 0, 0, 0);
    }
  };

  // NT: the wave's tiles that hold columns, known where this is compiled: with a branch around every product nothing overlaps
  // MASKED: some of the stage's keys are hidden from some columns.
  auto compute = [&](const char* stage, int blk, auto nt, auto masked) {
    constexpr int NT = decltype(nt)::value;
    constexpr bool MASKED = decltype(masked)::value;
    // ---- scores of a stage's keys x 16 NT columns
    f32x4 S[L::H][NT][2];
#pragma unroll
    for (int h = 0; h < L::H; ++h) {
      Frag a[2][QS];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < QS; ++s) a[t][s] = key_frag(stage + h * L::SLOT, t, s);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) S[h][ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < QS; ++s)
#pragma unroll
        for (int j = 0; j < (HALF ? 1 : 4); ++j)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
              if constexpr (HALF) S[h][ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][s].v, qf[ct][s].v, S[h][ct][t], 0, 0, 0);
              else S[h][ct][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[t][s].w[j]), __uint_as_float(qf[ct][s].w[j]), S[h][ct][t], 0, 0, 0);
            }
    }
    // ---- online softmax, one column a lane's; the maximum follows only when it has grown by more than 2^8, which keeps the sums
    // as far from overflow as they need be and leaves most stages without a rescaling
    if constexpr (MASKED) {
#pragma unroll
      for (int h = 0; h < L::H; ++h)
#pragma unroll
        for (int ct = 0; ct < NT; ++ct)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = key_at(blk, h, j);
            if (key < key_begin || key >= limit[ct]) S[h][ct][j >> 2][j & 3] = -INFINITY;
          }
    }
    float mx[NT];
    bool grown = false;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      mx[ct] = S[0][ct][0][0];
#pragma unroll
      for (int j = 1; j < 8 * L::H; ++j) mx[ct] = fmaxf(mx[ct], S[j >> 3][ct][j >> 2 & 1][j & 3]);
      mx[ct] = quad_max(mx[ct]) * scale_log2;
      grown |= mx[ct] > m[ct] + 8.f;
    }
    if (__any(grown)) {
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const float m_new = fmaxf(m[ct], mx[ct]);
        const float alpha = m[ct] == -INFINITY ? 0.f : fast_exp2(m[ct] - m_new);
        m[ct] = m_new;
        l[ct] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) O[ct][dt] *= alpha;
      }
    }
#pragma unroll
    for (int h = 0; h < L::H; ++h) {
      // the values of 32 keys, asked for before the weights are known
      constexpr int VF = HALF ? DT : 2 * DT;
      Frag va[VF];
#pragma unroll
      for (int f = 0; f < VF; ++f) va[f] = value_frag(stage + h * L::SLOT, f);
      float p[NT][8];
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const float base = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[ct][j] = fast_exp2(fmaf(S[h][ct][j >> 2][j & 3], scale_log2, -base));
          l[ct] += p[ct][j];
        }
      }
      if (MASKED && (blk < key_begin || blk + BLOCK_KEYS * (h + 1) > most)) {
#pragma unroll
        for (int f = 0; f < VF; ++f) clear_hidden(va[f], f, blk, h);
      }
      if constexpr (HALF) {
        Frag pb[NT];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct)
#pragma unroll
          for (int j = 0; j < 4; ++j) pb[ct].w[j] = pack_bf16(p[ct][2 * j], p[ct][2 * j + 1]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int ct = 0; ct < NT; ++ct) O[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[dt].v, pb[ct].v, O[ct][dt], 0, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int ct = 0; ct < NT; ++ct)
              O[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(va[2 * dt + (j >> 2)].w[j & 3]), p[ct][j], O[ct][dt], 0, 0, 0);
      }
    }
  };

  // one loop for each number of tiles a wave may have (waves of a workgroup meet at barriers, whichever loop they are in)
  auto walk = [&](auto nt) {
    int n = 0, stage = 0, fill = L::STAGES - 1;             // where stage n is, where stage n + STAGES - 1 goes
    auto step = [&](auto masked) {
      // stage n has landed for every wave, and nobody reads the one before any more
      if (n + L::STAGES - 1 < count) MIE_VMCNT((L::STAGES - 2) * L::H * L::EACH);
      else MIE_VMCNT(0);                                    // (the last ones may be shorter)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (n + L::STAGES - 1 < count) {
        issue_stage(n + L::STAGES - 1, fill);
        find_stage();
      }
      if constexpr (decltype(nt)::value > 0) compute(lds + stage * L::STAGE, blk0 + n * L::KEYS, nt, masked);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fill = stage;
      stage = stage + 1 < L::STAGES ? stage + 1 : 0;
      ++n;
    };
    const int whole = decltype(nt)::value > 0 ? (least - blk0) / L::KEYS : 0;      // stages before it end where every column sees them
    while (n < count) {
      if (n > 0 || blk0 >= key_begin)
        while (n < whole && n < count) step(std::false_type());
      if (n < count) step(std::true_type());
    }
  };
  if constexpr (L::APART) {
    if (apart) {
      constexpr int VF = HALF ? DT : 2 * DT;
      for (int n = 0; n < mine; ++n) {
        const int blk = blk1 + n * stride;
        if (L::SLOTS == 2 && n + 1 < mine) MIE_VMCNT(L::UNITS);        // the wave's next 32 keys may still be on their way
        else MIE_VMCNT(0);
        asm volatile("" ::: "memory");
        const char* slot = lds + (wave * L::SLOTS + (L::SLOTS == 2 ? n & 1 : 0)) * L::SLOT;
        Frag a[2][QS], va[VF];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int s = 0; s < QS; ++s) a[t][s] = key_frag(slot, t, s);
#pragma unroll
        for (int f = 0; f < VF; ++f) va[f] = value_frag(slot, f);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");              // read: the slot is free
        if (n + L::SLOTS < mine) {
          issue_own(L::SLOTS == 2 ? n & 1 : 0, next_own);
          next_own = find();
        }
        attend_one(a, va, blk);
      }
    }
    if (deal) {
      // ---- the waves' columns are the same: join them in the LDS, once nobody reads or writes a slot
      __shared__ float s_m[WAVES][16], s_l[WAVES][16];
      float* s_o = reinterpret_cast<float*>(lds);
      const float sum = quad_sum(l[0]);
      if (kb == 0) {
        s_m[wave][col] = m[0];
        s_l[wave][col] = sum;
      }
      __syncthreads();
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) M = fmaxf(M, s_m[w][col]);
      const float f = m[0] == -INFINITY ? 0.f : fast_exp2(m[0] - M);
      if (wave < L::SHARERS)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s_o[(wave * 16 + col) * (D + 1) + dt * 16 + 4 * kb + i] = m[0] == -INFINITY ? 0.f : O[0][dt][i] * f;
      __syncthreads();
      for (int e = threadIdx.x; e < 16 * D; e += WAVES * 64) {
        const int hc = e / D, d = e - hc * D, c = col0 + hc;
        if (c >= columns) break;
        float M1 = -INFINITY, total = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M1 = fmaxf(M1, s_m[w][hc]);
#pragma unroll
        for (int w = 0; w < L::SHARERS; ++w) {
          total += s_m[w][hc] == -INFINITY ? 0.f : fast_exp2(s_m[w][hc] - M1) * s_l[w][hc];
          y += s_o[(w * 16 + hc) * (D + 1) + d];
        }
        const int r = first_row + c / G, head = kvh * G + c % G;
        if (row_parts[r + 1] - row_parts[r] == 1) {
          const float sink = head_sinks ? head_sinks[head] * 1.4426950408889634f : sink_log2;
          const float all = total + (sink == -INFINITY ? 0.f : M1 == -INFINITY ? 1.f : fast_exp2(sink - M1));
          out[((size_t)r * Hq + head) * D + d] = from_float<T>(all == 0.f ? 0.f : y / all);
        } else {
          const size_t at = (size_t)(row_parts[r] + part) * Hq + head;
          o_part[at * D + d] = total == 0.f ? 0.f : y / total;
          if (d == 0) lse_part[at] = total == 0.f ? -INFINITY : M1 + log2f(total);
        }
      }
      return;
    }
  }
  if (!solo) {
    if (CT == 2 && tiles == 2) walk(std::integral_constant<int, CT>());
    else if (tiles > 0) walk(std::integral_constant<int, 1>());
    else walk(std::integral_constant<int, 0>());
  }

#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = col0 + ((solo ? 0 : wave * CT) + ct) * 16 + col;
    const float sum = quad_sum(l[ct]);
    if (c >= columns || (solo && ct > 0)) continue;
    const int r = first_row + c / G, head = kvh * G + c % G;
    const int slot = row_parts[r] + part;
    if (sum == 0.f) {       // a column that sees nothing, beside others that may see a value which is no number: 0 times that is in its O
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) O[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (row_parts[r + 1] - row_parts[r] == 1) {             // nothing to join: the result itself
      const float sink = head_sinks ? head_sinks[head] * 1.4426950408889634f : sink_log2;
      const float total = sum + (sink == -INFINITY ? 0.f : m[ct] == -INFINITY ? 1.f : fast_exp2(sink - m[ct]));
      const float inv = total == 0.f ? 0.f : 1.0f / total;
      T* o = out + ((size_t)r * Hq + head) * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
      {
        const f32x4 y = O[ct][dt] * inv;
        if constexpr (HALF) *reinterpret_cast<uint2*>(o + dt * 16 + 4 * kb) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        else *reinterpret_cast<f32x4*>(o + dt * 16 + 4 * kb) = y;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      float* o = o_part + ((size_t)slot * Hq + head) * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x4 y = O[ct][dt] * inv;
        *reinterpret_cast<f32x4*>(o + dt * 16 + 4 * kb) = y;
      }
      if (kb == 0) lse_part[(size_t)slot * Hq + head] = sum == 0.f ? -INFINITY : m[ct] + log2f(sum);
    }
  }
}

// The parts of a row and query head: weights from the log-sum-exps, then the parts' outputs, eight asked for together by each of the
// workgroup's waves, which take the parts in turn and meet in the LDS.
template <typename T>
__global__ void __launch_bounds__(WAVES * 64)
join_parts_kernel(const float* __restrict__ o_part, const float* __restrict__ lse_part, T* __restrict__ out,
                  const int* __restrict__ row_parts, int Hq, float sink_log2, const float* __restrict__ head_sinks) {
  constexpr int DL = (D + 63) / 64, AHEAD = 8;
  __shared__ float s_acc[WAVES][DL * 64], s_m[WAVES], s_w[WAVES];
  const int r = blockIdx.x / Hq, head = blockIdx.x - r * Hq, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int waves = blockDim.x >> 6;
  const int first = row_parts[r], n = row_parts[r + 1] - first;
  if (n == 1) return;                                       // written by its only item
  float acc[DL], W = 0.f, M = -INFINITY;
#pragma unroll
  for (int i = 0; i < DL; ++i) acc[i] = 0.f;
  for (int j0 = wave * AHEAD; j0 < n; j0 += waves * AHEAD) {
    float w[AHEAD], v[AHEAD][DL], most = M;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const size_t at = (size_t)(first + (j0 + j < n ? j0 + j : n - 1)) * Hq + head;
      w[j] = lse_part[at];
#pragma unroll
      for (int i = 0; i < DL; ++i) v[j][i] = o_part[at * D + (lane + 64 * i < D ? lane + 64 * i : 0)];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j0 + j >= n) w[j] = -INFINITY;
      most = fmaxf(most, w[j]);
    }
    const float f = M == -INFINITY ? 0.f : exp2f(M - most);
    M = most;
    W *= f;
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] *= f;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float x = w[j] == -INFINITY ? 0.f : exp2f(w[j] - M);
      W += x;
#pragma unroll
      for (int i = 0; i < DL; ++i) acc[i] = fmaf(x, v[j][i], acc[i]);
    }
  }
  if (waves > 1) {
    if (lane == 0) { s_m[wave] = M; s_w[wave] = W; }
#pragma unroll
    for (int i = 0; i < DL; ++i) s_acc[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    if (wave > 0) return;
    for (int w = 1; w < waves; ++w) {
      const float m2 = s_m[w], most = fmaxf(M, m2);
      const float f = M == -INFINITY ? 0.f : exp2f(M - most), g = m2 == -INFINITY ? 0.f : exp2f(m2 - most);
      M = most;
      W = W * f + s_w[w] * g;
#pragma unroll
      for (int i = 0; i < DL; ++i) acc[i] = acc[i] * f + s_acc[w][lane + 64 * i] * g;
    }
  }
  const float sink = head_sinks ? head_sinks[head] * 1.4426950408889634f : sink_log2;
  const float total = W + (sink == -INFINITY ? 0.f : M == -INFINITY ? 1.f : exp2f(sink - M));
  const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
  for (int i = 0; i < DL; ++i)
    if (lane + 64 * i < D) out[((size_t)r * Hq + head) * D + lane + 64 * i] = from_float<T>(acc[i] * inv);
}

MIE_EXPORT const char* shared_attention_last_error() { return g_mie_error; }
MIE_EXPORT int mie_shared_attention_head_dim() { return D; }

template <typename T, int CT>
static int launch_items(const void* q, long q_stride, const void* k_cache, const void* v_cache, void* out, float* o_part, float* lse_part,
                        const int* tables, int max_blocks, int pages, const int* positions, const int* items, int num_items, int whole_items,
                        const int* row_parts, int Hq, int Hkv, int page, float scale, float sink, const float* head_sinks, hipStream_t stream) {
  auto* kernel = shared_attention_kernel<T, CT>;
  constexpr int lds = Layout<T, CT>::LDS;
  if (lds > 65536 - 1024 && mie_allow_lds(reinterpret_cast<const void*>(kernel), lds, "shared_prefix_attention")) return -1;
  const int q_vec = ((uintptr_t)q & 15) == 0 && (q_stride * (long)sizeof(T)) % 16 == 0;
  constexpr int SOLO = Layout<T, CT>::SHARERS;
  const unsigned groups = whole_items + (num_items - whole_items + SOLO - 1) / SOLO;
  hipLaunchKernelGGL(kernel, dim3(groups * Hkv), dim3(WAVES * 64), lds, stream, (const T*)q, q_stride, q_vec,
                     (const T*)k_cache, (const T*)v_cache, (T*)out, o_part, lse_part, tables, max_blocks, pages, positions,
                     (const SharedItem*)items, num_items, whole_items, row_parts, Hq, Hkv, page, scale, sink, head_sinks);
  MIE_CHECK_LAUNCH("shared_prefix_attention");
  return 0;
}

// items [num_items, 8] (the first whole_items take a workgroup each, the others a wave each), row_parts [rows + 1]: the plan's; o_part [slots, Hq, D] and lse_part [slots, Hq] hold the partial results of rows
// with several parts (slot row_parts[r] + part).  most_parts: the largest number of parts a row has, or 1 if every row has exactly one.  scale, sink: in units of log2 e.
MIE_EXPORT int mie_shared_attention(const void* q, long q_stride, const void* k_cache, const void* v_cache, void* out, int dtype, float* o_part,
                                    float* lse_part, const int* tables, int max_blocks, int pages, const int* positions, int rows,
                                    const int* items, int num_items, int whole_items, int column_tiles, const int* row_parts, int most_parts, int Hq, int Hkv,
                                    int page, float scale_log2, float sink_log2, const float* head_sinks, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (Hkv < 1 || Hq < 1 || Hq % Hkv || page < 16 || page % 16 || page > 1 << 20 || max_blocks < 1 || pages < 1)
    MIE_FAIL("shared_prefix_attention: %d query heads, %d kv heads, pages of %d keys", Hq, Hkv, page);
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) MIE_FAIL("shared_prefix_attention: caches that do not begin on 16 bytes");
  if (!(scale_log2 > 0.f)) MIE_FAIL("shared_prefix_attention: the scale must be above 0");
  if ((long)num_items * Hkv > 0x7FFFFFFFL || (long)rows * Hq > 0x7FFFFFFFL) MIE_FAIL("shared_prefix_attention: too many items or rows");
  if (num_items > 0) {
    int rc;
#define MIE_ITEMS(T, CT) launch_items<T, CT>(q, q_stride, k_cache, v_cache, out, o_part, lse_part, tables, max_blocks, pages, positions, items, \
                                             num_items, whole_items, row_parts, Hq, Hkv, page, scale_log2, sink_log2, head_sinks, stream)
    const int most = dtype == MIE_BF16 ? MOST_TILES : 1;
    const int row_bytes = D * (dtype == MIE_BF16 ? 2 : 4);
    if (whole_items < 0 || whole_items > num_items || (whole_items < num_items && row_bytes % 64))
      MIE_FAIL("shared_prefix_attention: %d of %d items of a workgroup, heads of %d numbers", whole_items, num_items, D);
    if (column_tiles < 1 || column_tiles > most) MIE_FAIL("shared_prefix_attention: %d tiles of columns a wave, at most %d", column_tiles, most);
    if (dtype == MIE_BF16) rc = column_tiles == MOST_TILES ? MIE_ITEMS(bf16, MOST_TILES) : MIE_ITEMS(bf16, 1);
    else rc = MIE_ITEMS(float, 1);
    if (rc) return rc;
  }
  if (most_parts != 1) {
    const int waves = most_parts > 24 ? 4 : most_parts > 8 ? 2 : 1;
    if (dtype == MIE_BF16)
      hipLaunchKernelGGL(join_parts_kernel<bf16>, dim3((unsigned)rows * Hq), dim3(64 * waves), 0, stream, o_part, lse_part, (bf16*)out, row_parts, Hq,
                         sink_log2, head_sinks);
    else
      hipLaunchKernelGGL(join_parts_kernel<float>, dim3((unsigned)rows * Hq), dim3(64 * waves), 0, stream, o_part, lse_part, (float*)out, row_parts, Hq,
                         sink_log2, head_sinks);
    MIE_CHECK_LAUNCH("shared_prefix_attention");
  }
  return 0;
}
