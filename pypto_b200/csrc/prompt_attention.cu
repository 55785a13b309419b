// Attention over packed prompts: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that token i of a sequence sees, in one
// pass over the keys with a running maximum and sum.
//
// The query heads of a key head are rows of one matrix (row = token * group + head), so a work item is 256 rows of a sequence
// against its keys: two MMA tiles of 128 rows, two streams, and every K and V tile that is loaded serves both. A stream goes in
// steps of 64 keys. TMEM holds the scores of two steps of each stream, whose first half the probabilities overwrite as 16-bit
// values (the A operand of the value product from there), and both outputs; the scores of step i + 2 follow the value product of
// step i, so the softmax finds the next step's scores ready while the tensor pipe works on the ones before. Measured on 8192 tokens x
// 32 heads on 8 key heads of 128, causal: 452 to 470 us, 1170 to 1216 TFLOP/s (71 to 73 % of the GEMM's burst rate; under the power cap
// of a long run 521).
// Steps of 128 keys in one buffer, probabilities handed over by halves: the pipe waits for the softmax and the softmax for it, 497;
// scores and probabilities of 64 keys in columns of their own, two hand-overs a step: 505, where this had 485. What bounds it is shared
// memory, which delivers 128 bytes a cycle: score products of 64 keys take 48 cycles instead of 32, and without any softmax at all
// the kernel still takes 401 us.
// An item of at most 128 rows (a few tokens, single ones) has one tile; both streams take it, each with half of the keys, and the
// halves are merged at the end.
// Scores, maxima, sums and outputs are fp32. Probabilities alone are rounded to the rows' type, since the value product takes 16-bit
// operands; their sum is that of the unrounded ones. That adds a third to the error that rounding the output has in any case: bf16
// 0.0020 of the outputs' size from the definition in 64 bits, where fp32 throughout and one rounding has 0.0015; f16 0.00029 for 0.00021.
// Warps: 0 and 1 issue the MMAs of stream 0 and 1, 2 hands out items and loads K and V by TMA through a ring, 3 loads queries and
// mends the value tiles at a mask's edge, 4-7 and 8-11 are the softmax of stream 0 and 1, one thread a row.
#include "prompt_attention.cuh"
#include "sfa_common.cuh"

#include <climits>

namespace pto {
namespace {

constexpr int kThreads = 384;
constexpr int kBox = 16384;  // 128 rows of 128 bytes, 128-byte swizzle
constexpr uint32_t kTmemCols = 512;
constexpr float kLn2 = 0.693147180559945309f;

template <int DQK, int DV, bool F16>
struct Cfg {
  static constexpr int kSlotBoxes = DQK == 128 ? 2 : 1;  // boxes of 64 columns a ring slot holds
  static constexpr int kSlot = kSlotBoxes * kBox;
  static constexpr int kQ = DQK / 64 * kBox;
  static constexpr int kRing = (14 * kBox - 2 * kQ) / kSlot;  // 12, 5, 8 slots
  static constexpr int kK = DQK / 64 / kSlotBoxes, kV = DV / 64 / kSlotBoxes;  // slots of a K and of a V tile
  // From the slot that a stream waited for last to its next one: at most a K and a V tile of the other stream's between them. That is
  // within a lap, so what the loader had to see given back before it filled the last one covers the next one's use two laps ago, and
  // the barriers' parities, which tell even laps from odd ones, are unambiguous. (An item's first slot comes right behind the whole
  // item before, which the loader had issued when it gave out the item.)
  static_assert(kK + kV + 1 <= kRing, "a stream's next slot is more than a lap away");
  static constexpr int kStep = 64, kSteps = kPaKeys / kStep;  // keys of a step, steps of a tile
  static constexpr uint32_t kColO = 256;                      // first column of the outputs, behind two streams' two buffers of scores
  static constexpr uint32_t kFmt = F16 ? 0u : kABFmtBF16;
  static constexpr uint32_t kNonFinite = F16 ? 0x7c00u : 0x7f80u;  // exponent bits
  // f16 probabilities are kept away from its subnormal values: times 2^4 (a maximum that lags by 2^8 leaves them below 2^12)
  static constexpr float kBias = F16 ? 4.f : 0.f;
};
// Of eight pairs of probabilities, those whose exponentials the FMA pipe computes (8192 tokens, 0 to 3 of eight: 480, 462, 469, 472 us)
constexpr int kFmaPairs = 1;
constexpr float kLag = 8.f;  // a maximum is raised, and the output rescaled, once it is 2^8 behind
// A row's exponents are taken relative to its maximum's, rounded to fp32: fma(score, scale, -fl(maximum * scale)), exact but for a
// factor of 2^(up to half a step of the maximum's) in all of the row. From this exponent on that would be more than 2^(1/2), and soon
// more than fp32 or f16 probabilities hold: there the maximum is taken from the scores before they are scaled.
constexpr float kFar = 0x1p24f;

struct alignas(16) Item {
  int valid, dual;
  int q0, row0, rows;        // first token of the sequence, first row, rows of the item
  int k0, lk, seen;          // first key, keys; row r sees min(lk, seen + token) keys
  int begin[2], end[2];      // key tiles of the two streams
  int last[2];               // keys that some row of a stream sees
  int edge, keys;            // keys from `edge` on are hidden from some row, from `keys` on from all of them
  int head, slot;            // key head; slot of the partial result, -1: the item is whole
};

constexpr int kMaxRing = 12;
struct Ctl {
  unsigned long long full[kMaxRing], raw[kMaxRing], empty[kMaxRing];
  unsigned long long qfull[2], qempty[2], sfull[2][2], pfull[2][2], pfree[2], ofull[2], xfull, xempty, mfull[2], mempty[2], drain[2];
  Item item[2];
  int odd[2];  // values that are not finite were taken out of an item's tiles
  uint32_t tmem;
  int expired;
  PaHead head;
  union {  // a table of a tile a lane is in the loader's registers before the first item is known to anyone
    float2 xch[128];  // maximum and sum of stream 1
    PaTile tile[32];
  };
};
static_assert(sizeof(Ctl) <= 2048, "control block");
constexpr int kSmem = 1024 + 14 * kBox + 2048;

struct Ctx {
  Ctl* c;
  uint32_t q, ring, tmem;
};

// Waits for a phase. A wait that runs out sets the status and `expired`, after which no wait of the CTA waits any more and nothing
// more is loaded: the loops run to their ends on whatever is there. One test, without a vote, is all that a phase that is
// complete costs; callers of warp-wide instructions converge behind it.
__device__ __forceinline__ void wait_bar(Ctl* c, uint32_t bar, uint32_t parity, int32_t* status, int site) {
  if (mbar_try_wait(bar, parity)) return;
  const long long t0 = clock64();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(&c->expired)) return;
    if (clock64() - t0 > kWaitBudgetCycles) {
      c->expired = 1;
      set_status(status, PTO_ST_WAIT_EXPIRED, site, site);
      return;
    }
  }
}
__device__ __forceinline__ void wait_warp(Ctl* c, unsigned long long& bar, uint32_t parity, int32_t* status, int site) {
  wait_bar(c, smem_u32(&bar), parity, status, site);
  __syncwarp();
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ int row_token(const PaParams& p, int row) {
  return static_cast<int>((static_cast<unsigned long long>(static_cast<uint32_t>(row)) * p.group_mul) >> p.group_shift);
}
// keys that a row sees
__device__ __forceinline__ int row_limit(const PaParams& p, const Item& it, int row) {
  if (!p.causal) return it.lk;
  return min(max(it.seen + row_token(p, it.row0 + row), 0), it.lk);
}

// ---- the table of row tiles ----------------------------------------------------------------------------------
__device__ __forceinline__ int warp_inclusive(int x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
__device__ __forceinline__ int block_exclusive(int v, int* scan, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int x = warp_inclusive(v);
  __syncthreads();  // `scan` may still be read
  if (lane == 31) scan[warp] = x;
  __syncthreads();
  const int y = warp_inclusive(lane < warps ? scan[lane] : 0);
  *total = __shfl_sync(0xffffffffu, y, 31);
  const int before = __shfl_sync(0xffffffffu, y, max(warp - 1, 0));
  return (warp > 0 ? before : 0) + x - v;
}
__device__ __forceinline__ long long block_sum64(long long v, long long* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scan[warp] = v;
  __syncthreads();
  v = lane < warps ? scan[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int block_max(int v, int* scan) {  // (of values that are not negative)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) scan[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? scan[lane] : 0);
}

__device__ __forceinline__ void sequence(const PaParams& p, int i, int& q0, int& lq, int& k0, int& lk) {
  // offsets out of order or range leave a sequence empty or cut short (and set the status); none reaches outside the tensors
  q0 = min(max(__ldg(p.cu_q + i), 0), p.tq);
  lq = min(max(__ldg(p.cu_q + i + 1), q0), p.tq) - q0;
  k0 = min(max(__ldg(p.cu_k + i), 0), p.tk);
  lk = min(max(__ldg(p.cu_k + i + 1), k0), p.tk) - k0;
}
__device__ __forceinline__ void check_sequence(const PaParams& p, int i, int q0, int lq, int k0, int lk) {
  if (q0 != __ldg(p.cu_q + i) || q0 + lq != __ldg(p.cu_q + i + 1) || k0 != __ldg(p.cu_k + i) || k0 + lk != __ldg(p.cu_k + i + 1)) {
    set_status(p.status, PTO_ST_BAD_PAGE, i, 73);
  }
}
__device__ __forceinline__ int tile_keys(const PaParams& p, const PaTile& t) {  // key tiles
  const int rows = min(kPaRows, t.lq * p.group - t.row0);
  const int keys = p.causal ? min(max(t.lk - t.lq + 1 + row_token(p, t.row0 + rows - 1), 0), t.lk) : t.lk;
  return (keys + kPaKeys - 1) / kPaKeys;
}

constexpr int kBuckets = 256;
constexpr int kPieceCost = 4, kCutCost = 4;
struct PlanScratch {
  long long sum[32];
  int scan[32];
  int n[kPaSmallTiles];          // small tables: key tiles of a row tile; others: places of the buckets
  int first[kPaSmallTiles + 1];  // small tables: first row tile of a sequence
};
static_assert(kBuckets <= kPaSmallTiles, "buckets");

// Row tiles, longest first, and how many pieces each is cut into. Called by all threads of a block. `head`, `tile`, `first`: the
// table. `ctas`: CTAs that will work.
__device__ void build_table(const PaParams& p, PaHead* head, PaTile* tile, int* first, PlanScratch* s, int ctas) {
  const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  if (p.max_tiles <= kPaSmallTiles) first = s->first;  // (b is at most max_tiles)
  int total = 0;
  for (int base = 0; base < p.b; base += nt) {
    const int i = base + tid;
    int count = 0;
    if (i < p.b) {
      int q0, lq, k0, lk;
      sequence(p, i, q0, lq, k0, lk);
      check_sequence(p, i, q0, lq, k0, lk);
      count = static_cast<int>((static_cast<long long>(lq) * p.group + kPaRows - 1) / kPaRows);
    }
    int all;
    const int at = block_exclusive(count, s->scan, &all);
    if (i < p.b) first[i] = min(total + at, p.max_tiles);
    total = min(total + all, p.max_tiles);
  }
  __syncthreads();
  auto look = [&](int t) {
    int lo = 0, hi = p.b - 1;  // last sequence whose first tile is at most t (those without tiles share theirs with the next)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    PaTile x;
    sequence(p, lo, x.q0, x.lq, x.k0, x.lk);
    x.row0 = (t - first[lo]) * kPaRows;
    x.pieces = 1;
    x.piece = x.slot = 0;
    return x;
  };
  const bool small = total <= min(nt, kPaSmallTiles);
  PaTile mine;
  int n = 0, longest = 0;
  long long sum = 0;
  if (small) {
    if (tid < total) {
      mine = look(tid);
      sum = longest = n = tile_keys(p, mine);
      s->n[tid] = n;
    }
  } else {
    for (int t = tid; t < total; t += nt) {
      const int k = tile_keys(p, look(t));
      sum += k;
      longest = max(longest, k);
    }
  }
  sum = block_sum64(sum, s->sum) * p.hkv;
  longest = block_max(longest, s->scan);

  // Pieces of at most `piece` key tiles, every one of which costs a CTA about kPieceCost tiles' time beside its keys, and kCutCost more
  // where its results are partial. Where there are fewer items than CTAs (they go round, in order): the shortest pieces of which there
  // are no more than CTAs, or shorter ones in several rounds, whichever ends first. More items are handed out as CTAs become free: a
  // long piece at the end leaves the others idle. (16 sequences of 1 to 16384 keys x 8 heads: one round 117 us, thirds of a CTA's share 98, this 94.)
  int piece = max(longest, 1);
  if (p.slots > 0 && longest > kPaMinPiece) {
    const long long share = (sum + ctas - 1) / ctas;
    if (small) {
      const bool rounds = static_cast<long long>(total) * p.hkv <= ctas;
      const auto count = [&](int len, int& slots) {  // pieces of a head; called by a warp
        int all = 0, cut = 0;
        for (int t = lane; t < total; t += 32) {
          const int k = max((s->n[t] + len - 1) / len, 1);
          all += k;
          cut += k > 1 ? k : 0;
        }
        slots = __reduce_add_sync(0xffffffffu, cut);
        return __reduce_add_sync(0xffffffffu, all);
      };
      int lo = longest;
      if (rounds) {  // each warp counts for a length of its own
        int hi = longest, slots;
        lo = kPaMinPiece;  // (as long as the longest: one piece each, which fits)
        while (lo < hi) {
          const int mid = lo + (hi - lo) * warp / warps;
          const int all = count(mid, slots);
          __syncthreads();
          if (lane == 0) s->scan[warp] = all * p.hkv <= ctas ? mid : INT_MAX;
          __syncthreads();
          // the shortest that fits, and the longest below it that does not
          const int fits = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(lane < warps ? s->scan[lane] : INT_MAX)));
          const int mine_mid = lo + (hi - lo) * lane / warps;
          const int fails = static_cast<int>(__reduce_max_sync(0xffffffffu, lane < warps && s->scan[min(lane, warps - 1)] == INT_MAX ? mine_mid : 0));
          hi = min(hi, fits);
          lo = max(lo, min(fails + 1, hi));
        }
      }
      // 32 lengths from a quarter of a share to two, and the one above
      long long best = LLONG_MAX;
      for (int j = warp; j <= 32; j += warps) {
        const int len = j == 32 ? lo : static_cast<int>(max(static_cast<long long>(kPaMinPiece), share * (j + 4) / 16));
        if (len > longest) continue;
        int slots;
        const long long all = static_cast<long long>(count(len, slots)) * p.hkv;
        const long long cost = rounds ? (all + ctas - 1) / ctas * (len + kPieceCost + (slots > 0 ? kCutCost : 0)) * 2
                                      : 2 * (sum + all * kPieceCost + static_cast<long long>(slots) * p.hkv * kCutCost) / ctas + len;
        if (static_cast<long long>(slots) * p.hkv <= p.slots) best = min(best, cost << 24 | len);  // (below 2^24 tiles)
      }
      __syncthreads();
      if (lane == 0) s->sum[warp] = best;
      __syncthreads();
      for (int i = 0; i < warps; ++i) best = min(best, s->sum[i]);
      if (best != LLONG_MAX) piece = static_cast<int>(best & 0xffffff);
    } else {
      const int third = static_cast<int>(max((share + 2) / 3, static_cast<long long>(kPaMinPiece)));
      if (longest > 2 * third && 2 * sum / third <= p.slots) piece = third;
    }
  }

  if (small) {
    // Every thread counts the pieces before its tile's: no scan, and nothing of the table is read back.
    const auto pieces_of = [&](int k) { return max((k + piece - 1) / piece, 1); };
    if (tid < total) s->first[tid] = mine.pieces = pieces_of(n);  // (the sequences' first tiles have been looked up)
    __syncthreads();
    int rank = 0, before = 0, slots_before = 0, all = 0, cut = 0;
    for (int t = 0; t < total; ++t) {
      const int k = s->n[t], c = s->first[t], many = c > 1 ? c : 0;
      const bool ahead = k > n || (k == n && t < tid);
      rank += ahead;
      before += ahead ? c : 0;
      slots_before += ahead ? many : 0;
      all += c;
      cut += many > 0;  // (the longest come first, and so do those in pieces)
    }
    if (tid < total) {
      mine.piece = before;
      mine.slot = mine.pieces > 1 ? slots_before : -1;
      tile[rank] = mine;
    }
    if (tid == 0) *head = PaHead{total, all, 0, cut};
    __syncthreads();
    return;
  }
  int pieces_all = 0, slots_all = 0, cut = 0;  // cut: tiles up to the last one in pieces
  const float per = static_cast<float>(kBuckets - 1) / static_cast<float>(max(longest, 1));
  auto bucket = [&](int k) { return kBuckets - 1 - static_cast<int>(static_cast<float>(k) * per); };
  for (int i = tid; i < kBuckets; i += nt) s->n[i] = 0;
  __syncthreads();
  for (int t = tid; t < total; t += nt) atomicAdd(&s->n[min(max(bucket(tile_keys(p, look(t))), 0), kBuckets - 1)], 1);
  __syncthreads();
  int all;
  const int c = tid < kBuckets ? s->n[tid] : 0;
  const int at = block_exclusive(c, s->scan, &all);
  if (tid < kBuckets) s->n[tid] = at;
  __syncthreads();
  for (int t = tid; t < total; t += nt) {
    PaTile x = look(t);
    const int k = tile_keys(p, x);
    x.pieces = max((k + piece - 1) / piece, 1);
    tile[atomicAdd(&s->n[min(max(bucket(k), 0), kBuckets - 1)], 1)] = x;
  }
  __syncthreads();
  for (int base = 0; base < total; base += nt) {
    const int t = base + tid;
    const int c = t < total ? tile[t].pieces : 0;
    int all, all_slots;
    const int at = block_exclusive(c, s->scan, &all);
    const int at_slot = block_exclusive(c > 1 ? c : 0, s->scan, &all_slots);
    cut = max(cut, block_max(c > 1 ? t + 1 : 0, s->scan));
    if (t < total) {
      tile[t].piece = pieces_all + at;
      tile[t].slot = c > 1 ? slots_all + at_slot : -1;
    }
    pieces_all += all;
    slots_all += all_slots;
  }
  if (tid == 0) *head = PaHead{total, pieces_all, 0, cut};
  __syncthreads();
}

// The same for a table of at most 32 tiles that cannot be in pieces, by one warp without a barrier. (17 tokens x 8 heads: 10.2 us with the block's,
// 8.8 with this.) `mark`: 32 ints.
__device__ __forceinline__ void build_short_table(const PaParams& p, PaHead* head, PaTile* tile, int* mark) {
  const int lane = threadIdx.x & 31;
  PaTile x = {};
  int count = 0;
  mark[lane] = 0;
  if (lane < p.b) {  // (b is at most max_tiles)
    sequence(p, lane, x.q0, x.lq, x.k0, x.lk);
    check_sequence(p, lane, x.q0, x.lq, x.k0, x.lk);
    count = (x.lq * p.group + kPaRows - 1) / kPaRows;
  }
  const int end = warp_inclusive(count);
  const int total = min(__shfl_sync(0xffffffffu, end, 31), p.max_tiles), first = end - count;
  __syncwarp();
  if (count > 0 && first < 32) mark[first] = lane;
  __syncwarp();
  int of = mark[lane];  // the tile's sequence: the last one that begins at or before it
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, of, o);
    if (lane >= o) of = max(of, y);
  }
  x.row0 = (lane - __shfl_sync(0xffffffffu, first, of)) * kPaRows;
  x.q0 = __shfl_sync(0xffffffffu, x.q0, of);
  x.lq = __shfl_sync(0xffffffffu, x.lq, of);
  x.k0 = __shfl_sync(0xffffffffu, x.k0, of);
  x.lk = __shfl_sync(0xffffffffu, x.lk, of);
  const int n = lane < total ? tile_keys(p, x) : -1;
  int rank = 0;
  for (int t = 0; t < total; ++t) {
    const int k = __shfl_sync(0xffffffffu, n, t);
    rank += k > n || (k == n && t < lane);
  }
  x.pieces = 1;
  x.piece = rank;
  x.slot = -1;
  if (lane < total) tile[rank] = x;
  if (lane == 0) *head = PaHead{total, total, 0, 0};
}

__global__ void __launch_bounds__(1024) pa_plan_kernel(const PaParams p, int ctas) {
  __shared__ PlanScratch s;
  pdl_trigger();
  PaHead* head = reinterpret_cast<PaHead*>(p.tables);
  PaTile* tile = reinterpret_cast<PaTile*>(head + 1);
  build_table(p, head, tile, reinterpret_cast<int*>(tile + p.max_tiles), &s, ctas);
}

// Item number w of a table: sets of key heads one after the other, in each the pieces of all tiles with the set's heads side by side.
// Called by a converged warp; `own`: the lane's tile of a table of at most 32.
__device__ __forceinline__ Item find_item(const PaParams& p, const PaTile* tile, const PaTile& own, int tiles, int pieces, long long w) {
  Item it = {};
  if (w >= static_cast<long long>(pieces) * p.hkv) return it;
  const unsigned per_set = static_cast<unsigned>(pieces) * p.head_set;  // (pieces * heads: the host side refuses 2^31)
  const int set = static_cast<unsigned>(w) / per_set;
  const int rem = static_cast<unsigned>(w) - set * per_set;
  const int heads = min(p.head_set, p.hkv - set * p.head_set);
  const int which = rem / heads;
  it.head = set * p.head_set + rem - which * heads;
  // the last tile whose first piece is at most `which`: 32 probes a step, whole in the last one
  const int lane = threadIdx.x & 31;
  int lo = 0, n = tiles;
  while (n > 32) {
    const int step = (n + 31) / 32;
    const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && tile[lo + lane * step].piece <= which);
    const int last = 31 - __clz(below);  // (lane 0's holds always)
    lo += last * step;
    n = min(step, n - last * step);
  }
  PaTile t = own;
  if (tiles > 32 && lane < n) t = tile[lo + lane];
  const int at = 31 - __clz(__ballot_sync(0xffffffffu, lane < n && t.piece <= which));
  t.q0 = __shfl_sync(0xffffffffu, t.q0, at);
  t.lq = __shfl_sync(0xffffffffu, t.lq, at);
  t.k0 = __shfl_sync(0xffffffffu, t.k0, at);
  t.lk = __shfl_sync(0xffffffffu, t.lk, at);
  t.row0 = __shfl_sync(0xffffffffu, t.row0, at);
  t.pieces = __shfl_sync(0xffffffffu, t.pieces, at);
  t.piece = __shfl_sync(0xffffffffu, t.piece, at);
  t.slot = __shfl_sync(0xffffffffu, t.slot, at);
  const int part = which - t.piece;
  it.valid = 1;
  it.q0 = t.q0;
  it.row0 = t.row0;
  it.rows = min(kPaRows, t.lq * p.group - t.row0);
  it.k0 = t.k0;
  it.lk = t.lk;
  it.seen = t.lk - t.lq + 1;
  it.dual = it.rows <= 128;
  const int n_all = tile_keys(p, t);
  const int begin = static_cast<int>(static_cast<long long>(n_all) * part / t.pieces);
  const int end = static_cast<int>(static_cast<long long>(n_all) * (part + 1) / t.pieces);
  it.edge = row_limit(p, it, 0);
  it.keys = row_limit(p, it, it.rows - 1);
  it.last[0] = it.dual ? it.keys : row_limit(p, it, 127);
  it.last[1] = it.keys;
  if (it.dual) {
    const int mid = begin + (end - begin + 1) / 2;
    it.begin[0] = begin;
    it.end[0] = it.begin[1] = mid;
    it.end[1] = end;
  } else {
    it.begin[0] = it.begin[1] = begin;
    const int end0 = (it.last[0] + kPaKeys - 1) / kPaKeys;
    it.end[0] = max(min(end, end0), begin);
    it.end[1] = end;
  }
  it.slot = t.pieces > 1 ? (t.slot * p.hkv + it.head * t.pieces + part) : -1;
  return it;
}

// ---- roles -----------------------------------------------------------------------------------------------------
template <int R>
__device__ __forceinline__ void ring_at(uint32_t pos, uint32_t& slot, uint32_t& phase) {
  const uint32_t lap = pos / R;
  slot = pos - lap * R;
  phase = lap & 1;
}

// Ring positions of the key and value tiles of step k of a stream, counted from the item's first slot, in the order of the loads:
// two tiles: K(0) | V(0) K(1) | V(1) K(2) ... for both streams; one tile: K0(0) K1(0) | V0(0) K0(1) V1(0) K1(1) | ...
template <typename C>
__device__ __forceinline__ uint32_t v_position(bool dual, int s, int k, int n0, int n1) {
  if (!dual) return C::kK * (k + 1) + C::kV * k;
  if (s == 0) return C::kK * (k + 1 + min(k + 1, n1)) + C::kV * (k + min(k, n1));
  return C::kK * (min(k + 2, n0) + k + 1) + C::kV * (2 * k + 1);
}
template <typename C>
__device__ __forceinline__ uint32_t k_position(bool dual, int s, int k, int n0, int n1) {
  if (k == 0) return dual && s == 1 ? C::kK : 0;
  return v_position<C>(dual, s, k - 1, n0, n1) + C::kV;
}

// Steps of a stream: whole tiles, but for the last one's where no row sees the rest
template <typename C>
__device__ __forceinline__ int item_steps(const Item& it, int s) {
  const int begin = s == 0 ? it.begin[0] : it.begin[1], n = (s == 0 ? it.end[0] : it.end[1]) - begin;
  return max(0, min(n * C::kSteps, ((s == 0 ? it.last[0] : it.last[1]) - begin * kPaKeys + C::kStep - 1) / C::kStep));
}

// K and V tiles through the ring, and the items
template <typename C, bool kOwnTable>
__device__ __forceinline__ void role_load(const PaParams& p, const Ctx& x, const CUtensorMap* mk, const CUtensorMap* mv, PaHead* head,
                                          const PaTile* tile) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31;
  const int tiles = head->tiles, pieces = head->pieces;
  PaTile own = {};
  if (lane < tiles && tiles <= 32) own = tile[lane];
  uint32_t pos = 0;
  long long w = blockIdx.x;
  for (uint32_t n_item = 0;; ++n_item) {
    const uint32_t buf = n_item & 1;
    wait_warp(c, c->mempty[buf], ((n_item >> 1) & 1) ^ 1, p.status, 80);
    Item it = find_item(p, tile, own, tiles, pieces, w);
    if (*reinterpret_cast<volatile int*>(&c->expired)) it.valid = 0;
    it.valid = __shfl_sync(0xffffffffu, it.valid, 0);
    if (lane == 0) {
      c->item[buf] = it;
      mbar_arrive(smem_u32(&c->mfull[buf]));
    }
    if (!it.valid) break;
    int next = 0;
    if (lane == 0 && !kOwnTable) next = atomicAdd(&head->next, 1);  // (its answer is due at the end of the item)
    auto load = [&](int slots, const CUtensorMap* map, int key_tile, bool edge) {
      for (int i = 0; i < slots; ++i, ++pos) {
        uint32_t slot, phase;
        ring_at<C::kRing>(pos, slot, phase);
        wait_warp(c, c->empty[slot], phase ^ 1, p.status, 81);
        if (elect_one() && !*reinterpret_cast<volatile int*>(&c->expired)) {
          const uint32_t bar = smem_u32(edge ? &c->raw[slot] : &c->full[slot]), dst = x.ring + slot * C::kSlot;
          mbar_arrive_expect_tx(bar, C::kSlot);
#pragma unroll
          for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
            tma_load_3d(dst + bx * kBox, map, (i * C::kSlotBoxes + bx) * 64, it.head, it.k0 + key_tile * kPaKeys, bar);
          }
        }
        __syncwarp();
      }
    };
    const int n0 = it.end[0] - it.begin[0], n1 = it.end[1] - it.begin[1], n = max(n0, n1);
    auto key = [&](int s, int k) { load(C::kK, mk, it.begin[s] + k, false); };
    auto value = [&](int s, int k) {
      const int j = it.begin[s] + k;
      load(C::kV, mv, j, (j + 1) * kPaKeys > it.edge);
    };
    if (!it.dual) {  // both streams read stream 1's tiles
      if (n > 0) key(1, 0);
      for (int k = 0; k < n; ++k) {
        value(1, k);
        if (k + 1 < n) key(1, k + 1);
      }
    } else {
      if (n0 > 0) key(0, 0);
      if (n1 > 0) key(1, 0);
      for (int k = 0; k < n; ++k) {
        if (k < n0) value(0, k);
        if (k + 1 < n0) key(0, k + 1);
        if (k < n1) value(1, k);
        if (k + 1 < n1) key(1, k + 1);
      }
    }
    w = kOwnTable ? w + gridDim.x : static_cast<long long>(gridDim.x) + __shfl_sync(0xffffffffu, next, 0);
  }
  if (*reinterpret_cast<volatile int*>(&c->expired)) {  // copies in flight arrive before the CTA ends
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitBudgetCycles / 64) {}
  }
}

// a * 0 + b of pairs: not a number once a value was not finite
template <bool F16>
__device__ __forceinline__ uint32_t times_zero(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (F16) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(b));
  else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(b));
  return d;
}

// Queries of the item's tiles into shared memory; value tiles at the edge: keys that no row sees become zeros (they may be another
// sequence's, or anything), and of keys that some rows do not see, values that are not finite become zeros (0 * inf is not 0); the
// rows that do see them get them added at the end.
template <typename C, int DQK, int DV, bool F16>
__device__ __forceinline__ void role_queries(const PaParams& p, const Ctx& x, const CUtensorMap* mq) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31;
  uint32_t base = 0, raw_phase = 0;
  for (uint32_t n_item = 0;; ++n_item) {
    const uint32_t buf = n_item & 1;
    wait_warp(c, c->mfull[buf], (n_item >> 1) & 1, p.status, 82);
    if (*reinterpret_cast<volatile int*>(&c->expired)) break;
    const Item& it = c->item[buf];
    if (!it.valid) break;
    const bool dual = it.dual;
    if (lane == 0) c->odd[buf] = 0;
    const int q0 = it.q0, row0 = it.row0, rows = it.rows, head = it.head * p.group;
    if (p.q_map) {
      // rows are token-major, so a tile is a box of 128 / group tokens x group heads; what lies behind the sequence is not written
      const int token = q0 + row_token(p, row0);
      if (n_item > 0 && elect_one()) {  // into L2 while the tiles are still read
        for (int s = 0; s < (dual ? 1 : 2); ++s) {
#pragma unroll
          for (int ch = 0; ch < DQK / 64; ++ch) {
            asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(mq), "r"(ch * 64), "r"(head),
                         "r"(token + (s == 1 ? row_token(p, 128) : 0))
                         : "memory");
          }
        }
      }
      __syncwarp();
      for (int s = 0; s < 2; ++s) {
        if (n_item > 0) wait_warp(c, c->qempty[s], (n_item - 1) & 1, p.status, 83);
        if (elect_one() && !*reinterpret_cast<volatile int*>(&c->expired)) {
          const uint32_t bar = smem_u32(&c->qfull[s]);
          if (s == 1 && dual) {
            mbar_arrive(bar);
          } else {
            mbar_arrive_expect_tx(bar, C::kQ);
#pragma unroll
            for (int ch = 0; ch < DQK / 64; ++ch) {
              tma_load_3d(x.q + s * C::kQ + ch * kBox, mq, ch * 64, head, token + (s == 1 ? row_token(p, 128) : 0), bar);
            }
          }
        }
        __syncwarp();
      }
    } else {
      const int piece = lane & 7;
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + piece * 8;
      for (int s = 0; s < 2; ++s) {
        if (n_item > 0) wait_warp(c, c->qempty[s], (n_item - 1) & 1, p.status, 83);
        if (s == 0 || !dual) {
#pragma unroll 4
          for (int i = 0; i < 32; ++i) {
            const int r = i * 4 + (lane >> 3), row = s * 128 + r;
            const bool in = row < rows;
            const int token = row_token(p, row0 + (in ? row : 0));
            const int h = head + row0 + (in ? row : 0) - token * p.group;
            const uint16_t* src = q + static_cast<int64_t>(q0 + token) * p.q_token + h * p.q_head;
            const uint32_t dst = x.q + s * C::kQ + r * 128 + ((piece ^ (r & 7)) << 4);
#pragma unroll
            for (int ch = 0; ch < DQK / 64; ++ch) cp_async_16(dst + ch * kBox, src + ch * 64, in ? 16 : 0);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c->qfull[s]));
      }
    }

    const int b0 = it.begin[0], b1 = it.begin[1], n0 = it.end[0] - b0, n1 = it.end[1] - b1, n = max(n0, n1);
    const int edge = it.edge, keys = it.keys, first = edge / kPaKeys;  // first tile at the edge
    for (int k = max(0, min(first - b0, first - b1)); k < n; ++k) {
      for (int st = dual ? 0 : 1; st < 2; ++st) {
        const int j = (st == 0 ? b0 : b1) + k;
        if (k >= (st == 0 ? n0 : n1) || j < first) continue;
        const uint32_t at = base + v_position<C>(dual, st, k, n0, n1);
        for (int i = 0; i < C::kV; ++i) {
          uint32_t slot, phase;
          ring_at<C::kRing>(at + i, slot, phase);
          wait_warp(c, c->raw[slot], (raw_phase >> slot) & 1, p.status, 84);
          raw_phase ^= 1u << slot;
          // rows [from, keep) are looked at, rows from keep on cleared; a lane has 16 bytes of every fourth row
          const int from = max(edge - j * kPaKeys, 0), keep = min(max(keys - j * kPaKeys, 0), kPaKeys);
          const uint32_t mine = x.ring + slot * C::kSlot + (lane >> 3) * 128 + (lane & 7) * 16;
          const int r0 = lane >> 3;
          for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
            const uint32_t a = mine + bx * kBox;
            uint32_t seen = 0;
#pragma unroll 8
            for (int g = from >> 2; g < (keep + 3) >> 2; ++g) {
              const uint4 v = lds_v4u(a + g * 512);
              seen = times_zero<F16>(v.x, times_zero<F16>(v.y, times_zero<F16>(v.z, times_zero<F16>(v.w, seen))));
            }
            if ((seen & 0x7fff7fffu) != 0) {  // (rows below `from` or from keep on may have set it off)
              for (int g = from >> 2; g < (keep + 3) >> 2; ++g) {
                const int r = g * 4 + r0;
                if (r < from || r >= keep) continue;
                uint4 v = lds_v4u(a + g * 512);
                uint32_t* u = reinterpret_cast<uint32_t*>(&v);
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t lo = C::kNonFinite, hi = C::kNonFinite << 16;
                  if ((u[e] & lo) == lo) {
                    u[e] &= 0xffff0000u;
                    bad = true;
                  }
                  if ((u[e] & hi) == hi) {
                    u[e] &= 0xffffu;
                    bad = true;
                  }
                }
                if (bad) {
                  sts_v4u(a + g * 512, v);
                  c->odd[buf] = 1;
                }
              }
            }
            for (int g = keep >> 2; g < kPaKeys / 4; ++g) {
              if (g * 4 + r0 >= keep) sts_v4u(a + g * 512, make_uint4(0, 0, 0, 0));
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&c->full[slot]));
        }
      }
    }
    base += (dual ? n0 + n1 : n) * (C::kK + C::kV);
    if (lane == 0) mbar_arrive(smem_u32(&c->mempty[buf]));
  }
}

// The MMAs of one stream: S(0) S(1) | PV(0) S(2) | PV(1) S(3) ... One thread does all of it (with a converged warp that elects a lane
// for every batch of products 8192 tokens x 32 heads took 557 us instead of 505).
template <typename C, int DQK, int DV, int S>
__device__ __forceinline__ void role_mma(const PaParams& p, const Ctx& x) {
  Ctl* c = x.c;
  constexpr uint32_t kIdS = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 0, 128, C::kStep);
  constexpr uint32_t kIdO = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 1, 128, DV), kIdO64 = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 1, 128, 64);
  const uint32_t t_o = x.tmem + C::kColO + S * DV;
  const uint32_t sfull = smem_u32(&c->sfull[S][0]), pfree = smem_u32(&c->pfree[S]), empty = smem_u32(&c->empty[0]), full = smem_u32(&c->full[0]);
  const uint32_t pfull = smem_u32(&c->pfull[S][0]);
  const uint64_t k_desc = umma_desc_kmajor_sw128(x.ring), v_desc = desc_mnmajor_sw128(x.ring, kBox, 1024);
  uint32_t base = 0, ns = 0, np = 0;
  // A slot is free once both streams have read it; one that only this stream reads is given back twice. Before its next load is
  // waited for, the one before, maybe of the other stream alone, must have been given back: a barrier tells even laps from odd ones.
  auto loaded = [&](uint32_t at) {
    const uint32_t lap = at / C::kRing, slot = at - lap * C::kRing;
    if (lap > 0) wait_bar(c, empty + slot * 8, (lap - 1) & 1, p.status, 86);
    wait_bar(c, full + slot * 8, lap & 1, p.status, 87);
  };
  auto give_back = [&](uint32_t slot, bool alone) {
    tc_commit(empty + slot * 8);
    if (alone) tc_commit(empty + slot * 8);
  };
  for (uint32_t n_item = 0;; ++n_item) {
    const uint32_t buf = n_item & 1;
    wait_bar(c, smem_u32(&c->mfull[buf]), (n_item >> 1) & 1, p.status, 89);
    if (*reinterpret_cast<volatile int*>(&c->expired)) break;
    const Item it = c->item[buf];  // (in registers: under the products' reads a look into shared memory takes some 200 cycles)
    if (!it.valid) break;
    const bool dual = it.dual;
    const int n0 = it.end[0] - it.begin[0], n1 = it.end[1] - it.begin[1], n = item_steps<C>(it, S);
    const int q_tile = dual ? 0 : S;
    const uint64_t a = umma_desc_kmajor_sw128(x.q + q_tile * C::kQ);
    // (its own barrier as well, so that it is never more than a phase behind)
    wait_bar(c, smem_u32(&c->qfull[S]), n_item & 1, p.status, 90);
    if (q_tile != S) wait_bar(c, smem_u32(&c->qfull[q_tile]), n_item & 1, p.status, 90);
    auto queries_read = [&]() { tc_commit(smem_u32(&c->qempty[q_tile])); };
    auto score = [&](int i) {
      const int k = i / C::kSteps, h = i % C::kSteps;
      const bool last = h == C::kSteps - 1 || i + 1 == n, alone = dual || (S == 1 && k >= n0);
      const uint32_t at = base + k_position<C>(dual, S, k, n0, n1), t_s = x.tmem + S * 128 + (ns & 1) * 64;
#pragma unroll
      for (int j = 0; j < C::kK; ++j) {
        if (h == 0) loaded(at + j);
        const uint32_t slot = (at + j) % C::kRing;
        const uint64_t b = k_desc + (slot * (C::kSlot >> 4) + h * (C::kStep * 128 >> 4));
        tc_fence_after();
#pragma unroll
        for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            mma_f16_ss(t_s, a + ((j * C::kSlotBoxes + bx) * (kBox >> 4) + kk * 2), b + (bx * (kBox >> 4) + kk * 2), kIdS, (j | bx | kk) != 0);
          }
        }
        if (j == C::kK - 1) tc_commit(sfull + (ns & 1) * 8);
        if (last) give_back(slot, alone);
      }
      ++ns;
      if (i + 1 == n) queries_read();
    };
    if (n == 0) queries_read();
    if (S == 1) mbar_arrive(smem_u32(&c->qempty[dual ? 1 : 0]));  // the tile that it does not read
    for (int i = 0; i < 2 && i < n; ++i) score(i);
    for (int i = 0; i < n; ++i, ++np) {
      const int k = i / C::kSteps, h = i % C::kSteps;
      const uint32_t at = base + v_position<C>(dual, S, k, n0, n1), t_p = x.tmem + S * 128 + (np & 1) * 64;
      uint32_t slot[C::kV];
#pragma unroll
      for (int j = 0; j < C::kV; ++j) {
        slot[j] = (at + j) % C::kRing;
        if (h == 0) loaded(at + j);
      }
      wait_bar(c, pfull + (np & 1) * 8, (np >> 1) & 1, p.status, 88);
      tc_fence_after();
      // boxes of 64 value columns side by side: one product of dv columns, unless the ring wraps between them
      if (C::kV == 1 || slot[C::kV - 1] == slot[0] + C::kV - 1) {
        const uint64_t b = v_desc + (slot[0] * (C::kSlot >> 4) + h * (C::kStep * 128 >> 4));
#pragma unroll
        for (int kk = 0; kk < C::kStep / 16; ++kk) mma_f16_ts(t_o, t_p + kk * 8, b + kk * 128, kIdO, i > 0 || kk > 0);
      } else {
#pragma unroll
        for (int j = 0; j < C::kV; ++j) {
          const uint64_t b = v_desc + (slot[j] * (C::kSlot >> 4) + h * (C::kStep * 128 >> 4));
#pragma unroll
          for (int kk = 0; kk < C::kStep / 16; ++kk) mma_f16_ts(t_o + j * 64, t_p + kk * 8, b + kk * 128, kIdO64, i > 0 || kk > 0);
        }
      }
      tc_commit(pfree);
      if (i + 1 == n) tc_commit(smem_u32(&c->ofull[S]));
      if (h == C::kSteps - 1 || i + 1 == n) {
#pragma unroll
        for (int j = 0; j < C::kV; ++j) give_back(slot[j], dual || (S == 1 && k >= n0));
      }
      if (i + 2 < n) score(i + 2);
    }
    base += (dual ? n0 + n1 : max(n0, n1)) * (C::kK + C::kV);
    mbar_arrive(smem_u32(&c->mempty[buf]));
  }
  // what was issued completes before the CTA ends
  tc_commit(smem_u32(&c->drain[S]));
  wait_bar(c, smem_u32(&c->drain[S]), 0, p.status, 91);
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 u, v;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tadd.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// largest of three; a NaN stays one
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of a pair on the FMA pipe: x = n + f, |f| <= 1/2, n from the sum with 1.5 * 2^23; 2^f by the polynomial of degree four with
// p(0) = 1 and the smallest relative error on that interval (2.8e-6; computed by Lawson's iteration); n goes to the exponent. 0 for
// x <= -127. The exponential unit gives 16 values a clock and SM, so a tile's take as long as its products: a share of them goes
// this way.
template <int N, int M>
__device__ __forceinline__ void exp2_fma(float2 (&x)[M]) {  // of the first N pairs
  float2 t[N > 0 ? N : 1], y[N > 0 ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = make_float2(fmaxf(x[i].x, -127.f), fmaxf(x[i].y, -127.f));
    t[i] = add2(x[i], both(12582912.f));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = add2(x[i], fma2(t[i], both(-1.f), both(12582912.f)));
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fma2(x[i], both(0x1.3a02ccp-7f), both(0x1.c9fc46p-5f));
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fma2(x[i], y[i], both(0x1.ec0378p-3f));
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fma2(x[i], y[i], both(0x1.62e12cp-1f));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    y[i] = fma2(x[i], y[i], both(1.f));
    x[i].x = __int_as_float(__float_as_int(y[i].x) + (__float_as_int(t[i].x) << 23));
    x[i].y = __int_as_float(__float_as_int(y[i].y) + (__float_as_int(t[i].y) << 23));
  }
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (F16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}
template <bool F16>
__device__ __forceinline__ float to_float(uint16_t v) {
  if constexpr (F16) return __half2float(__ushort_as_half(v));
  else return __uint_as_float(static_cast<uint32_t>(v) << 16);
}

// `scale`: of an exponent of 2
__device__ __forceinline__ bool is_far(float m, float scale) { return m != -INFINITY && fabsf(m * scale) >= kFar; }
// What probabilities relative to a maximum m weigh beside those relative to a larger one (or the same)
__device__ __forceinline__ float weight_of(float m, float top, float scale) {
  if (m == -INFINITY) return 0.f;
  return ex2f(is_far(top, scale) ? (m - top) * scale : __fmul_rn(m, scale) - __fmul_rn(top, scale));
}
template <int DV>
__device__ __forceinline__ void rescale(uint32_t t_o, float f) {
#pragma unroll 1
  for (int i = 0; i < DV / 32; ++i) {
    uint32_t o[32];
    tmem_ld_32x32b_x32(t_o + i * 32, o);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    tmem_st_32x32b_x32(t_o + i * 32, o);
  }
}

// 32 bytes of a row: one store where they lie on a 32-byte boundary
__device__ __forceinline__ void store32(void* dst, const uint32_t (&w)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

template <typename C, int DV, bool F16>
__device__ __forceinline__ void role_softmax(const PaParams& p, const Ctx& x, int s) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31, r = threadIdx.x & 127;
  const uint32_t lanes = static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21;
  const uint32_t t_o = x.tmem + lanes + C::kColO + s * DV;
  const float sl = p.scale_log2;
  uint32_t ns = 0, no = 0, nx = 0;
  const uint32_t sfull = smem_u32(&c->sfull[s][0]), pfull = smem_u32(&c->pfull[s][0]);
  for (uint32_t n_item = 0;; ++n_item) {
    const uint32_t buf = n_item & 1;
    wait_warp(c, c->mfull[buf], (n_item >> 1) & 1, p.status, 92);
    if (*reinterpret_cast<volatile int*>(&c->expired)) break;
    const Item it = c->item[buf];
    if (!it.valid) break;
    const int n = item_steps<C>(it, s), key0 = (s == 0 ? it.begin[0] : it.begin[1]) * kPaKeys;
    const int row = (it.dual ? 0 : s * 128) + r;
    const bool mine = row < it.rows;
    const int limit = row_limit(p, it, mine ? row : it.rows - 1);
    const int sure = row_limit(p, it, it.dual ? 0 : s * 128);  // keys that all rows of the stream see
    float m = -INFINITY, l = 0.f;                              // maximum (of the scores as they are) and sum
    int k = 0;
    for (; k < n; ++k, ++ns) {
      const uint32_t t_s = x.tmem + lanes + s * 128 + (ns & 1) * 64;
      wait_bar(c, sfull + (ns & 1) * 8, (ns >> 1) & 1, p.status, 93);
      __syncwarp();
      tc_fence_after();
      if (key0 + (k + 1) * C::kStep > sure) {  // hidden keys: into the scores' columns, so that the way without any has no code for it
        const int left = limit - (key0 + k * C::kStep);
#pragma unroll 1
        for (int h = 0; h < C::kStep / 32; ++h) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_s + 32 * h, o);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 32 * h + i < left ? o[i] : 0xff800000u;
          tmem_st_32x32b_x32(t_s + 32 * h, o);
        }
        tc_wait_st();
      }
      uint32_t u[C::kStep / 32][32];
      float(&v)[C::kStep / 32][32] = reinterpret_cast<float(&)[C::kStep / 32][32]>(u);
#pragma unroll
      for (int h = 0; h < C::kStep / 32; ++h) tmem_ld_32x32b_x32(t_s + 32 * h, u[h]);
      tc_wait_ld();
      float top[C::kStep / 16];
#pragma unroll
      for (int h = 0; h < C::kStep / 16; ++h) {
        const float* w = &v[h >> 1][(h & 1) * 16];
        top[h] = max3(w[0], w[1], w[2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) top[h] = max3(top[h], w[e], w[e + 1]);
        top[h] = max3(top[h], w[15], h > 0 ? top[h - 1] : w[15]);
      }
      float t = top[C::kStep / 16 - 1];
      if (t == INFINITY) t = NAN;  // inf - inf: what the row comes to in any case
      if (k == 0) {
        if (__any_sync(0xffffffffu, is_far(t, sl))) break;
        m = t;
      } else {
        // the first maximum mostly stays good enough: the output is rescaled when it is more than 2^8 behind
        const bool raise = m == -INFINITY ? t != m : !((t - m) * sl <= kLag);
        if (__any_sync(0xffffffffu, raise)) {
          if (__any_sync(0xffffffffu, raise && is_far(t, sl))) break;
          const float f = raise ? (m == -INFINITY ? 0.f : ex2f((m - t) * sl)) : 1.f;
          m = raise ? t : m;
          l *= f;
          // the value product before (the one before that came ahead of these scores)
          wait_warp(c, c->pfree[s], (ns - 1) & 1, p.status, 94);
          tc_fence_after();
          rescale<DV>(t_o, f);
        }
      }
      const float2 shift = both(C::kBias - (m == -INFINITY ? 0.f : m * sl));
      float2 sum[2] = {both(0.f), both(0.f)};
#pragma unroll
      for (int h = 0; h < C::kStep / 32; ++h) {
        uint32_t w[16];
#pragma unroll
        for (int g = 0; g < 16; g += 8) {
          float2 y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = fma2(make_float2(v[h][2 * (g + e)], v[h][2 * (g + e) + 1]), both(sl), shift);
          exp2_fma<kFmaPairs>(y);
#pragma unroll
          for (int e = kFmaPairs; e < 8; ++e) y[e] = make_float2(ex2f(y[e].x), ex2f(y[e].y));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum[e & 1] = add2(sum[e & 1], y[e]);
            w[g + e] = pack16<F16>(y[e].x, y[e].y);
          }
        }
        tmem_st_32x32b_x16(t_s + h * 16, w);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + (ns & 1) * 8);
      l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
    }
    // The rest of an item in which a row of the warp has a maximum far from zero: the same steps, short rather than fast
    for (bool far = false; k < n; ++k, ++ns) {
      const uint32_t t_s = x.tmem + lanes + s * 128 + (ns & 1) * 64;
      wait_bar(c, sfull + (ns & 1) * 8, (ns >> 1) & 1, p.status, 93);
      __syncwarp();
      tc_fence_after();
      const int left = limit - (key0 + k * C::kStep);
      float t = -INFINITY;
#pragma unroll 1
      for (int h = 0; h < C::kStep / 32; ++h) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_s + 32 * h, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) t = max3(t, t, 32 * h + i < left ? __uint_as_float(o[i]) : -INFINITY);
      }
      if (t == INFINITY) t = NAN;
      const bool raise = m == -INFINITY ? t != m : !((t - m) * sl <= kLag);
      if (__any_sync(0xffffffffu, raise)) {
        const float f = raise ? (m == -INFINITY ? 0.f : ex2f((m - t) * sl)) : 1.f;
        m = raise ? t : m;
        l *= f;
        far = raise ? is_far(m, sl) : far;
        if (k > 0) {
          wait_warp(c, c->pfree[s], (ns - 1) & 1, p.status, 94);
          tc_fence_after();
          rescale<DV>(t_o, f);
        }
      }
      const float from = far ? m : 0.f, shift = C::kBias - (far || m == -INFINITY ? 0.f : m * sl);
#pragma unroll 1
      for (int h = 0; h < C::kStep / 32; ++h) {
        uint32_t o[32], w[16];
        tmem_ld_32x32b_x32(t_s + 32 * h, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float y[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int at = 2 * i + j;
            y[j] = 32 * h + at < left ? ex2f(fmaf(__uint_as_float(o[at]) - from, sl, shift)) : 0.f;
            l += y[j];
          }
          w[i] = pack16<F16>(y[0], y[1]);
        }
        tmem_st_32x32b_x16(t_s + h * 16, w);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + (ns & 1) * 8);
    }

    // ---- the item's output
    if (n > 0) {
      wait_warp(c, c->ofull[s], no & 1, p.status, 96);
      ++no;
      tc_fence_after();
    }
    if (it.dual && s == 1) {
      wait_warp(c, c->xempty, (nx & 1) ^ 1, p.status, 97);
      c->xch[r] = make_float2(m, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->xfull));
      // stream 0 reads this stream's output: the next item's first probabilities come after that
      wait_warp(c, c->xempty, nx & 1, p.status, 97);
      ++nx;
      if (lane == 0) mbar_arrive(smem_u32(&c->mempty[buf]));
      continue;
    }
    float f0 = 1.f, f1 = 0.f, top = m, all = l;
    bool two = false;
    if (it.dual) {
      wait_warp(c, c->xfull, nx & 1, p.status, 98);
      ++nx;
      const float2 o = c->xch[r];
      two = it.end[1] > it.begin[1];
      if (two) {
        const float best = fmaxf(top, o.x);
        f0 = weight_of(top, best, sl);
        f1 = weight_of(o.x, best, sl);
        all = l * f0 + o.y * f1;
        top = best;
      }
    }
    tc_fence_after();
    const bool odd = c->odd[buf] != 0;
    const int token = it.q0 + row_token(p, it.row0 + row);
    const int h = it.head * p.group + (it.row0 + row) - row_token(p, it.row0 + row) * p.group;
    const float inv = it.slot >= 0 ? 1.f : (all == 0.f ? 0.f : 1.f / all);
    f0 *= inv;
    f1 *= inv;
    uint8_t* dst = it.slot >= 0 ? reinterpret_cast<uint8_t*>(p.part_o + (static_cast<int64_t>(it.slot) * p.slot_rows + row) * DV)
                                : reinterpret_cast<uint8_t*>(reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + h * p.out_head);
    const bool any = __any_sync(0xffffffffu, mine);
#pragma unroll 1  // (code that runs once an item is kept small: it is fetched anew every time)
    for (int i = 0; any && i < DV / 32; ++i) {
      uint32_t a[32];
      float y[32];
      if (n > 0) {
        tmem_ld_32x32b_x32(t_o + i * 32, a);
        tc_wait_ld();
#pragma unroll
        for (int q = 0; q < 32; ++q) y[q] = __uint_as_float(a[q]) * f0;
      } else {
#pragma unroll
        for (int q = 0; q < 32; ++q) y[q] = 0.f;
      }
      if (two) {
        tmem_ld_32x32b_x32(t_o + DV + i * 32, a);
        tc_wait_ld();
#pragma unroll
        for (int q = 0; q < 32; ++q) y[q] = fmaf(__uint_as_float(a[q]), f1, y[q]);
      }
      if (odd && mine) {  // values that are not finite, of the keys at the edge that this row does see
        const int last = min(limit, it.end[1] * kPaKeys);
        const uint16_t* vp = reinterpret_cast<const uint16_t*>(p.v) + it.head * p.v_head + i * 32;
        for (int key = max(it.edge, it.begin[0] * kPaKeys); key < last; ++key) {
          const uint16_t* src = vp + static_cast<int64_t>(it.k0 + key) * p.v_token;
#pragma unroll
          for (int q = 0; q < 32; ++q) {
            const uint16_t bits = src[q];
            if ((bits & C::kNonFinite) == C::kNonFinite) y[q] += to_float<F16>(bits);
          }
        }
      }
      if (mine) {
        if (it.slot >= 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t w[8];
#pragma unroll
            for (int e2 = 0; e2 < 8; ++e2) w[e2] = __float_as_uint(y[8 * q + e2]);
            store32(dst + i * 128 + q * 32, w, true);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t w[8];
#pragma unroll
            for (int e2 = 0; e2 < 8; ++e2) w[e2] = pack16<F16>(y[16 * q + 2 * e2], y[16 * q + 2 * e2 + 1]);
            store32(dst + i * 64 + q * 32, w, p.out_wide);
          }
        }
      }
    }
    if (mine) {
      if (it.slot >= 0) {
        p.part_ml[static_cast<int64_t>(it.slot) * p.slot_rows + row] = make_float2(top, all);
      } else if (p.lse != nullptr) {
        p.lse[static_cast<int64_t>(h) * p.tq + token] = all == 0.f ? -INFINITY : (top * sl - C::kBias + log2f(all)) * kLn2;
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      if (it.dual) mbar_arrive(smem_u32(&c->xempty));
      mbar_arrive(smem_u32(&c->mempty[buf]));
    }
  }
}

// kOwnTable: every CTA builds the table. (Two kernels: with that code in the other's too, 4095 tokens x 128 heads of 192 took 416 us, not 371,
// and 8192 x 32 of 128 465, not 451.)
template <int DQK, int DV, bool F16, bool kOwnTable>
__global__ void __launch_bounds__(kThreads, 1)
pa_kernel(const PaParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
          const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<DQK, DV, F16>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t at = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (at - smem_u32(smem_raw));
  Ctl* c = reinterpret_cast<Ctl*>(base + 14 * kBox);
  const int warp = threadIdx.x >> 5;
  constexpr int kSetup = kThreads / 32 - 1;  // a warp that has nothing to look up for a short table: 900 cycles beside the first's loads
  if (threadIdx.x == kSetup * 32) {
    for (int i = 0; i < C::kRing; ++i) {
      mbar_init(smem_u32(&c->full[i]), 1);
      mbar_init(smem_u32(&c->raw[i]), 1);
      mbar_init(smem_u32(&c->empty[i]), 2);  // both streams
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&c->qfull[i]), 1);
      for (int j = 0; j < 2; ++j) {
        mbar_init(smem_u32(&c->sfull[i][j]), 1);
        mbar_init(smem_u32(&c->pfull[i][j]), 4);
      }
      mbar_init(smem_u32(&c->pfree[i]), 1);
      mbar_init(smem_u32(&c->ofull[i]), 1);
      mbar_init(smem_u32(&c->mfull[i]), 1);
      mbar_init(smem_u32(&c->mempty[i]), 11);  // warps 0, 1, 3 and the softmax's eight
      mbar_init(smem_u32(&c->drain[i]), 1);
    }
    mbar_init(smem_u32(&c->qempty[0]), 2);
    mbar_init(smem_u32(&c->qempty[1]), 1);
    mbar_init(smem_u32(&c->xfull), 4);
    mbar_init(smem_u32(&c->xempty), 4);
    c->expired = 0;
    fence_mbar_init();
  }
  if (warp == kSetup) {
    tmem_alloc(smem_u32(&c->tmem), kTmemCols);
    tmem_relinquish();
  } else if (warp == 2 && p.tk > 0 && elect_one()) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  uint8_t* table = p.tables + (kOwnTable ? blockIdx.x * p.table_stride : 0);
  PaHead* head = reinterpret_cast<PaHead*>(table);
  PaTile* tile = reinterpret_cast<PaTile*>(head + 1);
  if constexpr (kOwnTable) {
    // (scratch in the ring: the barrier at its end and the fence come before the first copy into it)
    const bool here = p.max_tiles <= 32;  // (in the workspace the merge alone reads it: 16 tokens x 8 heads 88.1 -> 87.5 us)
    if (here) head = &c->head, tile = c->tile;
    if (here && p.slots == 0) {
      if (warp == 0) build_short_table(p, head, tile, reinterpret_cast<int*>(base));
    } else {
      build_table(p, head, tile, nullptr, reinterpret_cast<PlanScratch*>(base), gridDim.x);
    }
    if (here && p.slots > 0 && blockIdx.x == 0 && warp == 0) {
      if ((threadIdx.x & 31) < head->tiles) reinterpret_cast<PaTile*>(table + sizeof(PaHead))[threadIdx.x & 31] = tile[threadIdx.x & 31];
      if (elect_one()) *reinterpret_cast<PaHead*>(table) = *head;
    }
  } else {
    pdl_wait();
  }
  pdl_trigger();
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const Ctx x{c, at, at + 2 * C::kQ, c->tmem};
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp < 2) {
      if (elect_one()) {
        if (warp == 0) role_mma<C, DQK, DV, 0>(p, x);
        else role_mma<C, DQK, DV, 1>(p, x);
      }
      __syncwarp();
    } else if (warp == 2) role_load<C, kOwnTable>(p, x, &map_k, &map_v, head, tile);
    else role_queries<C, DQK, DV, F16>(p, x, &map_q);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    role_softmax<C, DV, F16>(p, x, warp < 8 ? 0 : 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSetup) {
    tc_fence_after();
    tmem_dealloc(c->tmem, kTmemCols);
  }
}

// Tiles in several pieces: their partial results, weighted by 2^(maximum - the largest maximum). A warp a row.
template <int DV, bool F16>
__global__ void __launch_bounds__(256) pa_merge_kernel(const PaParams p) {
  constexpr int kPer = DV / 32;
  pdl_wait();
  const PaHead* head = reinterpret_cast<const PaHead*>(p.tables);
  const PaTile* tile = reinterpret_cast<const PaTile*>(head + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (p.slot_rows + 7) / 8;  // of rows: a block takes eight
  const long long work = static_cast<long long>(head->cut) * p.hkv * chunks;
  for (long long w = blockIdx.x; w < work; w += gridDim.x) {
    const long long item = w / chunks;
    const PaTile t = tile[item / p.hkv];
    if (t.pieces <= 1) continue;
    const int hk = static_cast<int>(item % p.hkv);
    const int rows = min(kPaRows, t.lq * p.group - t.row0);
    const int64_t slot = static_cast<int64_t>(t.slot) * p.hkv + hk * t.pieces;
    if (const int row = static_cast<int>(w - item * chunks) * 8 + warp; row < rows) {
      // a lane's piece, of the first 32: its maximum and sum
      const float2 own = lane < t.pieces ? p.part_ml[(slot + lane) * p.slot_rows + row] : make_float2(-INFINITY, 0.f);
      float top = own.x;
      for (int i = lane + 32; i < t.pieces; i += 32) top = fmaxf(top, p.part_ml[(slot + i) * p.slot_rows + row].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float y[kPer] = {}, all = 0.f;
      for (int i0 = 0; i0 < t.pieces; i0 += 32) {
        float2 ml = own;
        if (i0 > 0) ml = i0 + lane < t.pieces ? p.part_ml[(slot + i0 + lane) * p.slot_rows + row] : make_float2(-INFINITY, 0.f);
        const float weight = weight_of(ml.x, top, p.scale_log2);  // (0: it has seen no key)
        all += ml.x == -INFINITY ? 0.f : ml.y * weight;
        const int n = min(32, t.pieces - i0);
        const float* src = p.part_o + ((slot + i0) * p.slot_rows + row) * DV + lane * kPer;
        const int64_t step = static_cast<int64_t>(p.slot_rows) * DV;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const float f = __shfl_sync(0xffffffffu, weight, i);
          float v[kPer];
          if constexpr (kPer == 4) {
            const float4 q = __ldcg(reinterpret_cast<const float4*>(src + i * step));
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
          } else {
            const float2 q = __ldcg(reinterpret_cast<const float2*>(src + i * step));
            v[0] = q.x, v[1] = q.y;
          }
#pragma unroll
          for (int e = 0; e < kPer; ++e) y[e] = f != 0.f ? fmaf(v[e], f, y[e]) : y[e];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      const float inv = all == 0.f ? 0.f : 1.f / all;
      const int tok = row_token(p, t.row0 + row);
      const int h = hk * p.group + t.row0 + row - tok * p.group;
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (t.q0 + tok) * p.out_token + h * p.out_head + lane * kPer;
      if constexpr (kPer == 4) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<F16>(y[0] * inv, y[1] * inv), pack16<F16>(y[2] * inv, y[3] * inv));
      } else {
        *reinterpret_cast<uint32_t*>(dst) = pack16<F16>(y[0] * inv, y[1] * inv);
      }
      if (lane == 0 && p.lse != nullptr) {
        p.lse[static_cast<int64_t>(h) * p.tq + t.q0 + tok] = all == 0.f ? -INFINITY : (top * p.scale_log2 - Cfg<128, DV, F16>::kBias + log2f(all)) * kLn2;
      }
    }
  }
}

template <int DQK, int DV, bool F16>
cudaError_t launch(const PaParams& p, const void* tmap_q, const void* tmap_k, const void* tmap_v, int ctas, cudaStream_t stream) {
  const auto kernel = p.self_plan ? pa_kernel<DQK, DV, F16, true> : pa_kernel<DQK, DV, F16, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  if (!p.self_plan) {
    pa_plan_kernel<<<1, p.max_tiles <= kPaSmallTiles ? kPaSmallTiles : 1024, 0, stream>>>(p, ctas);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    count_launch();
  }
  e = launch_maybe_pdl(kernel, dim3(ctas), dim3(kThreads), kSmem, stream, !p.self_plan, p,
                       *reinterpret_cast<const CUtensorMap*>(tmap_q), *reinterpret_cast<const CUtensorMap*>(tmap_k), *reinterpret_cast<const CUtensorMap*>(tmap_v));
  if (e != cudaSuccess) return e;
  count_launch();
  if (p.slots > 0) {
    e = launch_maybe_pdl(pa_merge_kernel<DV, F16>, dim3(ctas * 5), dim3(256), 0, stream, true, p);
    count_launch();
  }
  return e;
}

}  // namespace

cudaError_t launch_prompt_attention(const PaParams& p, int dqk, int dv, int dtype, const void* tmap_q, const void* tmap_k,
                                    const void* tmap_v, int ctas, cudaStream_t stream) {
  const bool f16 = dtype == PTO_DT_F16;
#define PA_LAUNCH(a, b)                                                          \
  if (dqk == a && dv == b) {                                                     \
    return f16 ? launch<a, b, true>(p, tmap_q, tmap_k, tmap_v, ctas, stream)     \
               : launch<a, b, false>(p, tmap_q, tmap_k, tmap_v, ctas, stream);   \
  }
  PA_LAUNCH(64, 64)
  PA_LAUNCH(128, 128)
  PA_LAUNCH(192, 128)
#undef PA_LAUNCH
  return cudaErrorInvalidValue;
}

}  // namespace pto
