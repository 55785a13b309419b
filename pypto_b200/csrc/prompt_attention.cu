// Attention over packed prompts: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that token i of a sequence sees, in one
// pass over the keys with a running maximum and sum.
//
// The query heads of a key head are rows of one matrix (row = token * group + head), so a work item is 256 rows of a sequence
// against its keys: two MMA tiles of 128 rows, and every K and V tile that is loaded serves both. TMEM holds the scores of both
// tiles (2 x 128 columns) and both outputs (2 x dv); probabilities overwrite their scores as 16-bit values and are the A operand
// of the value product from there. While the softmax of one tile runs, the tensor pipe works for the other:
//   S0(0) S1(0) | PV0(0) S0(1) PV1(0) S1(1) | PV0(1) S0(2) ...
// An item of at most 128 rows (a few tokens, single ones) has one tile; both streams take it, each with half of the keys, and the
// halves are merged at the end.
// Warps: 0 issues MMAs, 1 hands out items and loads K and V by TMA through a ring, 2 and 3 load queries and mend the value tiles at
// a mask's edge, 4-7 and 8-11 are the softmax of stream 0 and 1, one thread a row.
#include "prompt_attention.cuh"
#include "sfa_common.cuh"

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
  static constexpr uint32_t kFmt = F16 ? 0u : kABFmtBF16;
  static constexpr uint32_t kNonFinite = F16 ? 0x7c00u : 0x7f80u;  // exponent bits
  // f16 probabilities are kept away from its subnormal values: times 2^4 (a maximum that lags by 2^8 leaves them below 2^12)
  static constexpr float kBias = F16 ? 4.f : 0.f;
};
constexpr float kLag = 8.f;  // a maximum is raised, and the output rescaled, once it is 2^8 behind

struct Item {
  int valid, dual;
  int q0, row0, rows;        // first token of the sequence, first row, rows of the item
  int k0, lk, seen;          // first key, keys; row r sees min(lk, seen + token) keys
  int begin[2], end[2];      // key tiles of the two streams
  int edge, keys;            // keys from `edge` on are hidden from some row, from `keys` on from all of them
  int head, slot;            // key head; slot of the partial result, -1: the item is whole
};

constexpr int kMaxRing = 12;
struct Ctl {
  unsigned long long full[kMaxRing], raw[kMaxRing], empty[kMaxRing];
  unsigned long long qfull[2], qempty, sfull[2], pfull[2], ofull[2], xfull, xempty, mfull[2], mempty[2], drain;
  Item item[2];
  int odd[2][2];  // values that are not finite were taken out of an item's tiles (by warp 2, by warp 3)
  uint32_t tmem;
  int scan[32];
  float2 xch[128];  // maximum and sum of stream 1
};
static_assert(sizeof(Ctl) <= 2048, "control block");
constexpr int kSmem = 1024 + 14 * kBox + 2048;

struct Ctx {
  Ctl* c;
  uint32_t q, ring, tmem;
};

__device__ __forceinline__ bool wait_bar(const unsigned long long& bar, uint32_t parity, int32_t* status, int site) {
  if (mbar_wait_spin(smem_u32(&bar), parity)) return true;
  set_status(status, PTO_ST_WAIT_EXPIRED, site, site);
  return false;
}
__device__ __forceinline__ bool wait_warp(const unsigned long long& bar, uint32_t parity, int32_t* status, int site) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, status, site));
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
__device__ __forceinline__ int block_exclusive(int v, int* scan, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // `scan` may still be read
  if (lane == 31) scan[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < warps; ++i) {
    before += i < warp ? scan[i] : 0;
    all += scan[i];
  }
  *total = all;
  return before + x - v;
}
__device__ __forceinline__ long long block_sum64(long long v, long long* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scan[warp] = v;
  __syncthreads();
  long long s = 0;
  for (int i = 0; i < warps; ++i) s += scan[i];
  return s;
}
__device__ __forceinline__ int block_max(int v, int* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scan[warp] = v;
  __syncthreads();
  int m = scan[0];
  for (int i = 1; i < warps; ++i) m = max(m, scan[i]);
  return m;
}

__device__ __forceinline__ void sequence(const PaParams& p, int i, int& q0, int& lq, int& k0, int& lk) {
  // offsets out of order or range leave a sequence empty or cut short (and set the status); none reaches outside the tensors
  q0 = min(max(__ldg(p.cu_q + i), 0), p.tq);
  lq = min(max(__ldg(p.cu_q + i + 1), q0), p.tq) - q0;
  k0 = min(max(__ldg(p.cu_k + i), 0), p.tk);
  lk = min(max(__ldg(p.cu_k + i + 1), k0), p.tk) - k0;
}
__device__ __forceinline__ int tile_keys(const PaParams& p, const PaTile& t) {  // key tiles
  const int rows = min(kPaRows, t.lq * p.group - t.row0);
  const int keys = p.causal ? min(max(t.lk - t.lq + 1 + row_token(p, t.row0 + rows - 1), 0), t.lk) : t.lk;
  return (keys + kPaKeys - 1) / kPaKeys;
}

constexpr int kBuckets = 256;
struct PlanScratch {
  long long sum[32];
  int scan[32];
  int n[kPaSmallTiles];  // small tables: key tiles of a row tile; others: places of the buckets
};
static_assert(kBuckets <= kPaSmallTiles, "buckets");

// Row tiles, longest first, and how many pieces each is cut into. Called by all threads of a block. `head`, `tile`, `first`: the
// table. `ctas`: CTAs that will work.
__device__ void build_table(const PaParams& p, PaHead* head, PaTile* tile, int* first, PlanScratch* s, int ctas) {
  const int nt = blockDim.x, tid = threadIdx.x;
  int total = 0;
  for (int base = 0; base < p.b; base += nt) {
    const int i = base + tid;
    int count = 0;
    if (i < p.b) {
      int q0, lq, k0, lk;
      sequence(p, i, q0, lq, k0, lk);
      if (q0 != __ldg(p.cu_q + i) || q0 + lq != __ldg(p.cu_q + i + 1) || k0 != __ldg(p.cu_k + i) || k0 + lk != __ldg(p.cu_k + i + 1)) {
        set_status(p.status, PTO_ST_BAD_PAGE, i, 73);
      }
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

  // Pieces of at most `piece` key tiles. Fewer items than CTAs: the shortest pieces that are no more than CTAs. More: a CTA's share
  // in four, so that the last ones to finish are not far apart (the partial results of a piece cost about a tile's time).
  int piece = max(longest, 1);
  if (p.slots > 0 && longest > kPaMinPiece) {
    if (static_cast<long long>(total) * p.hkv <= ctas && small) {
      int lo = kPaMinPiece, hi = longest;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const long long all = block_sum64((n + mid - 1) / mid + (tid < total && n == 0), s->sum);
        if (all * p.hkv <= ctas) hi = mid;
        else lo = mid + 1;
      }
      piece = lo;
    } else {
      const long long share = (sum + 4 * ctas - 1) / (4 * ctas);
      if (longest > 2 * share) piece = static_cast<int>(max(share, static_cast<long long>(kPaMinPiece)));
    }
  }

  if (piece < longest) {  // (the workspace is counted so that they fit)
    const int k = (n + piece - 1) / piece;
    const long long slots = small ? block_sum64(k > 1 ? k : 0, s->sum) * p.hkv : 2 * sum / piece;
    if (slots > p.slots) piece = longest;
  }

  int pieces_all = 0, slots_all = 0;
  if (small) {
    if (tid < total) s->n[tid] = n;
    __syncthreads();
    if (tid < total) {
      int rank = 0;
      for (int t = 0; t < total; ++t) rank += s->n[t] > n || (s->n[t] == n && t < tid);
      mine.pieces = max((n + piece - 1) / piece, 1);
      tile[rank] = mine;
    }
  } else {
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
  }
  __syncthreads();
  for (int base = 0; base < total; base += nt) {
    const int t = base + tid;
    const int c = t < total ? tile[t].pieces : 0;
    int all, all_slots;
    const int at = block_exclusive(c, s->scan, &all);
    const int at_slot = block_exclusive(c > 1 ? c : 0, s->scan, &all_slots);
    if (t < total) {
      tile[t].piece = pieces_all + at;
      tile[t].slot = c > 1 ? slots_all + at_slot : -1;
    }
    pieces_all += all;
    slots_all += all_slots;
  }
  if (tid == 0) *head = PaHead{total, pieces_all, 0, 0};
  __syncthreads();
}

__global__ void __launch_bounds__(1024) pa_plan_kernel(const PaParams p, int ctas) {
  __shared__ PlanScratch s;
  pdl_trigger();
  PaHead* head = reinterpret_cast<PaHead*>(p.tables);
  PaTile* tile = reinterpret_cast<PaTile*>(head + 1);
  build_table(p, head, tile, reinterpret_cast<int*>(tile + p.max_tiles), &s, ctas);
}

// Item number w of a table: sets of key heads one after the other, in each the pieces of all tiles with the set's heads side by side.
// Called by a converged warp.
__device__ __forceinline__ Item find_item(const PaParams& p, const PaTile* tile, int tiles, int pieces, long long w) {
  Item it = {};
  if (w >= static_cast<long long>(pieces) * p.hkv) return it;
  const long long per_set = static_cast<long long>(pieces) * p.head_set;
  const int set = static_cast<int>(w / per_set);
  const int rem = static_cast<int>(w - set * per_set);  // (below pieces * heads: the host side refuses 2^31)
  const int heads = min(p.head_set, p.hkv - set * p.head_set);
  const int which = rem / heads;
  it.head = set * p.head_set + rem - which * heads;
  // the last tile whose first piece is at most `which`: 32 probes a step
  const int lane = threadIdx.x & 31;
  int lo = 0, n = tiles;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int probe = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && tile[probe].piece <= which);
    const int last = 31 - __clz(below);  // (lane 0's holds always)
    lo += last * step;
    n = min(step, n - last * step);
  }
  const PaTile t = tile[lo];
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
  if (it.dual) {
    const int mid = begin + (end - begin + 1) / 2;
    it.begin[0] = begin;
    it.end[0] = it.begin[1] = mid;
    it.end[1] = end;
  } else {
    it.begin[0] = it.begin[1] = begin;
    const int end0 = (row_limit(p, it, 127) + kPaKeys - 1) / kPaKeys;
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

// Ring position of the value tile of step k of a stream, counted from the item's first slot (the order that the loads are in)
template <typename C>
__device__ __forceinline__ uint32_t v_position(const Item& it, int s, int k, int n0, int n1) {
  if (!it.dual) return C::kK * (k + 1) + C::kV * k;
  if (s == 0) return C::kK * (k + 1 + min(k + 1, n1)) + C::kV * (k + min(k, n1));
  return C::kK * (min(k + 2, n0) + k + 1) + C::kV * (2 * k + 1);
}

// K and V tiles through the ring, and the items
template <typename C, int DQK, int DV>
__device__ __forceinline__ void role_load(const PaParams& p, const Ctx& x, const CUtensorMap* mk, const CUtensorMap* mv, PaHead* head,
                                          const PaTile* tile) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31;
  const int tiles = head->tiles, pieces = head->pieces;
  uint32_t pos = 0;
  bool ok = true;
  long long w = blockIdx.x;
  for (uint32_t n_item = 0; ok; ++n_item) {
    const uint32_t buf = n_item & 1;
    ok = wait_warp(c->mempty[buf], ((n_item >> 1) & 1) ^ 1, p.status, 80);
    if (!ok) break;
    const Item it = find_item(p, tile, tiles, pieces, w);
    if (lane == 0) {
      c->item[buf] = it;
      mbar_arrive(smem_u32(&c->mfull[buf]));
    }
    if (!it.valid) break;
    int next = 0;
    if (lane == 0 && !p.self_plan) next = atomicAdd(&head->next, 1);  // (its answer is due at the end of the item)
    auto load = [&](int slots, int cols, const CUtensorMap* map, int key_tile, bool edge) {
      for (int i = 0; i < slots && ok; ++i, ++pos) {
        uint32_t slot, phase;
        ring_at<C::kRing>(pos, slot, phase);
        ok = wait_warp(c->empty[slot], phase ^ 1, p.status, 81);
        if (!ok) return;
        if (elect_one()) {
          const uint32_t bar = smem_u32(edge ? &c->raw[slot] : &c->full[slot]), dst = x.ring + slot * C::kSlot;
          mbar_arrive_expect_tx(bar, C::kSlot);
#pragma unroll
          for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                    dst + bx * kBox),
                "l"(map), "r"((i * C::kSlotBoxes + bx) * 64), "r"(it.head), "r"(it.k0 + key_tile * kPaKeys), "r"(bar)
                : "memory");
          }
        }
        __syncwarp();
      }
    };
    const int n0 = it.end[0] - it.begin[0], n1 = it.end[1] - it.begin[1], n = max(n0, n1);
    auto key = [&](int s, int k) { load(C::kK, DQK, mk, it.begin[s] + k, false); };
    auto value = [&](int s, int k) {
      const int j = it.begin[s] + k;
      load(C::kV, DV, mv, j, (j + 1) * kPaKeys > it.edge);
    };
    if (!it.dual) {  // both streams read stream 1's tiles
      if (n > 0) key(1, 0);
      for (int k = 0; k < n && ok; ++k) {
        value(1, k);
        if (k + 1 < n) key(1, k + 1);
      }
    } else {
      if (n0 > 0) key(0, 0);
      if (n1 > 0) key(1, 0);
      for (int k = 0; k < n && ok; ++k) {
        if (k < n0) value(0, k);
        if (k + 1 < n0) key(0, k + 1);
        if (k < n1) value(1, k);
        if (k + 1 < n1) key(1, k + 1);
      }
    }
    w = p.self_plan ? w + gridDim.x : static_cast<long long>(gridDim.x) + __shfl_sync(0xffffffffu, next, 0);
  }
  // whoever gave up: copies in flight arrive before the CTA ends
  if (!ok) {
    for (uint32_t i = pos > C::kRing ? pos - C::kRing : 0; i < pos; ++i) {
      uint32_t slot, phase;
      ring_at<C::kRing>(i, slot, phase);
      const long long t0 = clock64();
      while (!mbar_test_wait(smem_u32(&c->full[slot]), phase) && clock64() - t0 < kWaitBudgetCycles / 16) {}
    }
  }
}

// Queries of the item's tile into shared memory; value tiles at the edge: keys that no row sees become zeros (they may be another
// sequence's, or anything), and of keys that some rows do not see, values that are not finite become zeros (0 * inf is not 0); the
// rows that do see them get them added at the end.
template <typename C, int DQK, int DV, typename T>
__device__ __forceinline__ void role_queries(const PaParams& p, const Ctx& x, int s) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31;
  uint32_t base = 0, edges = 0, raw_phase = 0;
  bool ok = true;
  for (uint32_t n_item = 0; ok; ++n_item) {
    const uint32_t buf = n_item & 1;
    ok = wait_warp(c->mfull[buf], (n_item >> 1) & 1, p.status, 82);
    if (!ok) break;
    const Item it = c->item[buf];
    if (!it.valid) break;
    if (lane == 0) c->odd[buf][s] = 0;
    if (n_item > 0) ok = wait_warp(c->qempty, (n_item - 1) & 1, p.status, 83);
    if (!ok) break;
    if (s == 0 || !it.dual) {
      const int piece = lane & 7;
      const T* q = reinterpret_cast<const T*>(p.q) + piece * 8;
#pragma unroll 4
      for (int i = 0; i < 32; ++i) {
        const int r = i * 4 + (lane >> 3), row = s * 128 + r;
        const bool in = row < it.rows;
        const int token = row_token(p, it.row0 + (in ? row : 0));
        const int h = it.head * p.group + it.row0 + (in ? row : 0) - token * p.group;
        const T* src = q + static_cast<int64_t>(it.q0 + token) * p.q_token + h * p.q_head;
        const uint32_t dst = x.q + s * C::kQ + r * 128 + ((piece ^ (r & 7)) << 4);
#pragma unroll
        for (int ch = 0; ch < DQK / 64; ++ch) cp_async_16(dst + ch * kBox, src + ch * 64, in ? 16 : 0);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&c->qfull[s]));

    const int n0 = it.end[0] - it.begin[0], n1 = it.end[1] - it.begin[1], n = max(n0, n1);
    const int first = it.edge / kPaKeys;  // tile
    for (int k = max(0, min(first - it.begin[0], first - it.begin[1])); k < n && ok; ++k) {
      for (int st = it.dual ? 0 : 1; st < 2 && ok; ++st) {
        const int j = it.begin[st] + k;
        if (k >= (st == 0 ? n0 : n1) || j < first) continue;
        const uint32_t at = base + v_position<C>(it, st, k, n0, n1);
        for (int i = 0; i < C::kV; ++i, ++edges) {
          uint32_t slot, phase;
          ring_at<C::kRing>(at + i, slot, phase);
          const uint32_t rp = (raw_phase >> slot) & 1;
          raw_phase ^= 1u << slot;
          if ((edges & 1) != static_cast<uint32_t>(s)) continue;
          ok = wait_warp(c->raw[slot], rp, p.status, 84);
          if (!ok) break;
          const int from = max(it.edge - j * kPaKeys, 0), keep = it.keys - j * kPaKeys;
          bool odd = false;
          for (int r = (from & ~3) + (lane >> 3); r < 128; r += 4) {
            if (r < from) continue;
#pragma unroll
            for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
              const uint32_t a = x.ring + slot * C::kSlot + bx * kBox + r * 128 + (lane & 7) * 16;
              if (r >= keep) {
                sts_v4u(a, make_uint4(0, 0, 0, 0));
              } else {
                uint4 v = lds_v4u(a);
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
                  sts_v4u(a, v);
                  odd = true;
                }
              }
            }
          }
          if (odd) c->odd[buf][s] = 1;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&c->full[slot]));
        }
      }
    }
    base += (it.dual ? n0 + n1 : n) * (C::kK + C::kV);
    if (lane == 0) mbar_arrive(smem_u32(&c->mempty[buf]));
  }
}

template <typename C, int DQK, int DV>
__device__ __forceinline__ void role_mma(const PaParams& p, const Ctx& x) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31;
  constexpr uint32_t kIdS = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 0, 128, kPaKeys);
  uint32_t pos = 0, np[2] = {0, 0};
  bool ok = true;
  auto score = [&](int s, int q_tile, uint32_t at, bool last_use) {
    const uint64_t a = umma_desc_kmajor_sw128(x.q + q_tile * C::kQ);
#pragma unroll
    for (int i = 0; i < C::kK; ++i) {
      uint32_t slot, phase;
      ring_at<C::kRing>(at + i, slot, phase);
      if (!wait_warp(c->full[slot], phase, p.status, 85)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t b = umma_desc_kmajor_sw128(x.ring + slot * C::kSlot);
#pragma unroll
        for (int bx = 0; bx < C::kSlotBoxes; ++bx) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            mma_f16_ss(x.tmem + s * 128, a + ((i * C::kSlotBoxes + bx) * (kBox >> 4) + kk * 2), b + (bx * (kBox >> 4) + kk * 2), kIdS,
                       (i | bx | kk) != 0);
          }
        }
        if (last_use) tc_commit(smem_u32(&c->empty[slot]));
        if (i == C::kK - 1) tc_commit(smem_u32(&c->sfull[s]));
      }
      __syncwarp();
    }
    return true;
  };
  auto value = [&](int s, uint32_t at, bool first, bool last, bool last_use) {
    if (!wait_warp(c->pfull[s], np[s] & 1, p.status, 86)) return false;
    ++np[s];
    const uint32_t d = x.tmem + 256 + s * 128, a = x.tmem + s * 128;
    uint32_t slot[C::kV], phase;
#pragma unroll
    for (int i = 0; i < C::kV; ++i) {
      ring_at<C::kRing>(at + i, slot[i], phase);
      if (!wait_warp(c->full[slot[i]], phase, p.status, 87)) return false;
    }
    tc_fence_after();
    if (elect_one()) {
      // boxes of 64 value columns side by side: one product of dv columns, unless the ring wraps between them
      const bool joined = C::kV == 1 || slot[C::kV - 1] == slot[0] + C::kV - 1;
      if (joined) {
        constexpr uint32_t id = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 1, 128, DV);
        const uint64_t b = desc_mnmajor_sw128(x.ring + slot[0] * C::kSlot, kBox, 1024);
#pragma unroll
        for (int kk = 0; kk < kPaKeys / 16; ++kk) mma_f16_ts(d, a + kk * 8, b + kk * 128, id, !first || kk > 0);
      } else {
        constexpr uint32_t id = umma_idesc(kCFmtF32, C::kFmt, C::kFmt, 0, 1, 128, 64);
#pragma unroll
        for (int i = 0; i < C::kV; ++i) {
          const uint64_t b = desc_mnmajor_sw128(x.ring + slot[i] * C::kSlot, kBox, 1024);
#pragma unroll
          for (int kk = 0; kk < kPaKeys / 16; ++kk) mma_f16_ts(d + i * 64, a + kk * 8, b + kk * 128, id, !first || kk > 0);
        }
      }
      if (last_use) {
#pragma unroll
        for (int i = 0; i < C::kV; ++i) tc_commit(smem_u32(&c->empty[slot[i]]));
      }
      if (last) tc_commit(smem_u32(&c->ofull[s]));
    }
    __syncwarp();
    return true;
  };
  for (uint32_t n_item = 0; ok; ++n_item) {
    const uint32_t buf = n_item & 1;
    ok = wait_warp(c->mfull[buf], (n_item >> 1) & 1, p.status, 88);
    if (!ok) break;
    const Item it = c->item[buf];
    if (!it.valid) break;
    const bool dual = it.dual;
    const int n0 = it.end[0] - it.begin[0], n1 = it.end[1] - it.begin[1], n = max(n0, n1);
    uint32_t k_next = 0, v_now = 0;
    // slots in the order of the loads; in an item of two tiles stream 1 reads what stream 0 has read, and frees it
    auto take = [&](int slots) {
      const uint32_t at = pos;
      pos += slots;
      return at;
    };
    ok = wait_warp(c->qfull[0], n_item & 1, p.status, 89) && wait_warp(c->qfull[1], n_item & 1, p.status, 90);
    if (ok && n0 > 0) {
      k_next = take(C::kK);
      ok = score(0, 0, k_next, dual);
    }
    if (ok && n1 > 0) ok = score(1, dual ? 0 : 1, !dual && n0 > 0 ? k_next : take(C::kK), true);
    if (ok && n <= 1 && elect_one()) tc_commit(smem_u32(&c->qempty));
    __syncwarp();
    for (int k = 0; k < n && ok; ++k) {
      if (k < n0) {
        v_now = take(C::kV);
        ok = value(0, v_now, k == 0, k + 1 == n0, dual);
        if (ok && k + 1 < n0) {
          k_next = take(C::kK);
          ok = score(0, 0, k_next, dual);
        }
      }
      if (ok && k < n1) {
        ok = value(1, !dual && k < n0 ? v_now : take(C::kV), k == 0, k + 1 == n1, true);
        if (ok && k + 1 < n1) ok = score(1, dual ? 0 : 1, !dual && k + 1 < n0 ? k_next : take(C::kK), true);
      }
      // the queries have been read once the last scores are there
      if (ok && k + 2 == n && elect_one()) tc_commit(smem_u32(&c->qempty));
      __syncwarp();
    }
    if (lane == 0) mbar_arrive(smem_u32(&c->mempty[buf]));
  }
  // what was issued completes before the CTA ends
  if (elect_one()) tc_commit(smem_u32(&c->drain));
  __syncwarp();
  wait_warp(c->drain, 0, p.status, 91);
}

__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {  // (x, y) = (x, y) * a + b
  asm("{\n\t.reg .b64 v, s, t;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmov.b64 t, {%3, %3};\n\t"
      "fma.rn.f32x2 v, v, s, t;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 v, s;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tadd.rn.f32x2 v, v, s;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
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

template <typename C, int DV, bool F16>
__device__ __forceinline__ void role_softmax(const PaParams& p, const Ctx& x, int s) {
  Ctl* c = x.c;
  const int lane = threadIdx.x & 31, r = threadIdx.x & 127;
  const uint32_t lanes = static_cast<uint32_t>((threadIdx.x >> 5) & 3) << 21;
  const uint32_t t_s = x.tmem + lanes + s * 128, t_o = x.tmem + lanes + 256 + s * 128;
  const float sl = p.scale_log2;
  uint32_t ns = 0, no[2] = {0, 0}, nx = 0;
  bool ok = true;
  for (uint32_t n_item = 0; ok; ++n_item) {
    const uint32_t buf = n_item & 1;
    ok = wait_warp(c->mfull[buf], (n_item >> 1) & 1, p.status, 92);
    if (!ok) break;
    const Item& it = c->item[buf];
    if (!it.valid) break;
    const int begin = it.begin[s], n = it.end[s] - begin, n1 = it.end[1] - it.begin[1];
    const int row = (it.dual ? 0 : s * 128) + r;
    const bool mine = row < it.rows;
    const int limit = row_limit(p, it, mine ? row : it.rows - 1);
    const int sure = row_limit(p, it, it.dual ? 0 : s * 128);  // keys that all rows of the stream see
    float m = -INFINITY, l = 0.f;                              // maximum (of the scores as they are) and sum
    for (int k = 0; k < n; ++k, ++ns) {
      ok = wait_warp(c->sfull[s], ns & 1, p.status, 93);
      if (!ok) break;
      tc_fence_after();
      uint32_t u[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_s + i * 32, u[i]);
      tc_wait_ld();
      float(&v)[4][32] = reinterpret_cast<float(&)[4][32]>(u);
      const int j = begin + k;
      if ((j + 1) * kPaKeys > sure) {
        const int left = limit - j * kPaKeys;
#pragma unroll
        for (int i = 0; i < 128; ++i) v[i >> 5][i & 31] = i < left ? v[i >> 5][i & 31] : -INFINITY;
      }
      float top[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top[i] = v[i][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top[i] = fmaxf(top[i], v[i][e]);
      }
      const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (k == 0) {
        m = t;
      } else {
        // the first tile's maximum mostly stays good enough: the output is rescaled when it is more than 2^8 behind
        const bool raise = (t - m) * sl > kLag || (m == -INFINITY && t > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? (m == -INFINITY ? 0.f : ex2f((m - t) * sl)) : 1.f;
          m = raise ? t : m;
          l *= f;
          // (the scores of this tile are complete, so the value product before them is)
#pragma unroll
          for (int i = 0; i < DV / 32; ++i) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + i * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st_32x32b_x32(t_o + i * 32, o);
          }
        }
      }
      const float shift = C::kBias - (m == -INFINITY ? 0.f : m * sl);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float& a = v[2 * h + (e >> 4)][(2 * e) & 31];
          float& b = v[2 * h + (e >> 4)][(2 * e + 1) & 31];
          fma2(a, b, sl, shift);
          a = ex2f(a);
          b = ex2f(b);
          add2(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], a, b);
          w[e] = pack16<F16>(a, b);
        }
        tmem_st_32x32b_x32(t_s + h * 32, w);
      }
      l += (sum[0] + sum[2]) + (sum[1] + sum[3]);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->pfull[s]));
    }
    if (!ok) break;

    // ---- the item's output
    const int n_other = n1;
    if (s == 0 && !it.dual && n1 > 0) ++no[1];  // (another stream's phase that is not waited for here)
    if (n > 0) {
      ok = wait_warp(c->ofull[s], no[s] & 1, p.status, 94);
      ++no[s];
      if (!ok) break;
    }
    const float e = m * sl;  // exponent of the maximum
    if (it.dual && s == 1) {
      ok = wait_warp(c->xempty, (nx & 1) ^ 1, p.status, 95);
      if (!ok) break;
      c->xch[r] = make_float2(n > 0 ? e : -INFINITY, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->xfull));
      // stream 0 reads this stream's output: the next item's first probabilities come after that
      ok = wait_warp(c->xempty, nx & 1, p.status, 96);
      ++nx;
      if (lane == 0) mbar_arrive(smem_u32(&c->mempty[buf]));
      continue;
    }
    float f0 = 1.f, f1 = 0.f, top = n > 0 ? e : -INFINITY, all = l;
    bool two = false;
    if (it.dual) {
      ok = wait_warp(c->xfull, nx & 1, p.status, 97);
      ++nx;
      if (ok && n_other > 0) {
        ok = wait_warp(c->ofull[1], no[1] & 1, p.status, 98);
        ++no[1];
      }
      if (!ok) break;
      const float2 o = c->xch[r];
      two = n_other > 0;
      if (two) {
        const float best = fmaxf(top, o.x);
        f0 = top == -INFINITY ? 0.f : ex2f(top - best);
        f1 = o.x == -INFINITY ? 0.f : ex2f(o.x - best);
        all = l * f0 + o.y * f1;
        top = best;
      }
    }
    tc_fence_after();
    const bool odd = (c->odd[buf][0] | c->odd[buf][1]) != 0;
    const int token = it.q0 + row_token(p, it.row0 + row);
    const int h = it.head * p.group + (it.row0 + row) - row_token(p, it.row0 + row) * p.group;
    const float inv = it.slot >= 0 ? 1.f : (all == 0.f ? 0.f : 1.f / all);
    f0 *= inv;
    f1 *= inv;
#pragma unroll
    for (int i = 0; i < DV / 32; ++i) {
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
        tmem_ld_32x32b_x32(t_o + 128 + i * 32, a);
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
          float* dst = p.part_o + (static_cast<int64_t>(it.slot) * p.slot_rows + row) * DV + i * 32;
#pragma unroll
          for (int q = 0; q < 32; q += 4) *reinterpret_cast<float4*>(dst + q) = make_float4(y[q], y[q + 1], y[q + 2], y[q + 3]);
        } else {
          uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + h * p.out_head + i * 32;
#pragma unroll
          for (int q = 0; q < 32; q += 8) {
            *reinterpret_cast<uint4*>(dst + q) = make_uint4(pack16<F16>(y[q], y[q + 1]), pack16<F16>(y[q + 2], y[q + 3]),
                                                            pack16<F16>(y[q + 4], y[q + 5]), pack16<F16>(y[q + 6], y[q + 7]));
          }
        }
      }
    }
    if (mine) {
      if (it.slot >= 0) {
        p.part_ml[static_cast<int64_t>(it.slot) * p.slot_rows + row] = make_float2(top, all);
      } else if (p.lse != nullptr) {
        p.lse[static_cast<int64_t>(h) * p.tq + token] = all == 0.f ? -INFINITY : (top - C::kBias + log2f(all)) * kLn2;
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

template <int DQK, int DV, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
pa_kernel(const PaParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<DQK, DV, F16>;
  using T = uint16_t;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t at = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (at - smem_u32(smem_raw));
  Ctl* c = reinterpret_cast<Ctl*>(base + 14 * kBox);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kRing; ++i) {
      mbar_init(smem_u32(&c->full[i]), 1);
      mbar_init(smem_u32(&c->raw[i]), 1);
      mbar_init(smem_u32(&c->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&c->qfull[i]), 1);
      mbar_init(smem_u32(&c->sfull[i]), 1);
      mbar_init(smem_u32(&c->pfull[i]), 4);
      mbar_init(smem_u32(&c->ofull[i]), 1);
      mbar_init(smem_u32(&c->mfull[i]), 1);
      mbar_init(smem_u32(&c->mempty[i]), 11);  // warps 0, 2, 3 and the softmax's eight
    }
    mbar_init(smem_u32(&c->qempty), 1);
    mbar_init(smem_u32(&c->xfull), 4);
    mbar_init(smem_u32(&c->xempty), 4);
    mbar_init(smem_u32(&c->drain), 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&c->tmem), kTmemCols);
    tmem_relinquish();
  } else if (warp == 1 && p.tk > 0 && elect_one()) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  uint8_t* table = p.tables + (p.self_plan ? blockIdx.x * p.table_stride : 0);
  PaHead* head = reinterpret_cast<PaHead*>(table);
  PaTile* tile = reinterpret_cast<PaTile*>(head + 1);
  if (p.self_plan) {
    // (scratch in the ring: the barrier at its end and the fence come before the first copy into it)
    build_table(p, head, tile, reinterpret_cast<int*>(tile + p.max_tiles), reinterpret_cast<PlanScratch*>(base), gridDim.x);
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
    if (warp == 0) role_mma<C, DQK, DV>(p, x);
    else if (warp == 1) role_load<C, DQK, DV>(p, x, &map_k, &map_v, head, tile);
    else role_queries<C, DQK, DV, T>(p, x, warp - 2);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    role_softmax<C, DV, F16>(p, x, warp < 8 ? 0 : 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(c->tmem, kTmemCols);
  }
}

// Tiles in several pieces: their partial results, weighted by exp2(maximum - the largest maximum). A warp a row.
template <int DV, bool F16>
__global__ void __launch_bounds__(256) pa_merge_kernel(const PaParams p) {
  constexpr int kPer = DV / 32;
  pdl_wait();
  const PaHead* head = reinterpret_cast<const PaHead*>(p.tables);
  const PaTile* tile = reinterpret_cast<const PaTile*>(head + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long work = static_cast<long long>(head->tiles) * p.hkv;
  for (long long w = blockIdx.x; w < work; w += gridDim.x) {
    const PaTile t = tile[w / p.hkv];
    if (t.pieces <= 1) continue;
    const int hk = static_cast<int>(w % p.hkv);
    const int rows = min(kPaRows, t.lq * p.group - t.row0);
    const int64_t slot = static_cast<int64_t>(t.slot) * p.hkv + hk * t.pieces;
    for (int row = warp; row < rows; row += 8) {
      float top = -INFINITY;
      for (int i = lane; i < t.pieces; i += 32) top = fmaxf(top, p.part_ml[(slot + i) * p.slot_rows + row].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float y[kPer] = {}, all = 0.f;
#pragma unroll 4
      for (int i = 0; i < t.pieces; ++i) {
        const float2 ml = p.part_ml[(slot + i) * p.slot_rows + row];
        if (ml.x == -INFINITY) continue;
        const float f = ex2f(ml.x - top);
        all += ml.y * f;
        const float* src = p.part_o + ((slot + i) * p.slot_rows + row) * DV + lane * kPer;
        if constexpr (kPer == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          y[0] = fmaf(v.x, f, y[0]);
          y[1] = fmaf(v.y, f, y[1]);
          y[2] = fmaf(v.z, f, y[2]);
          y[3] = fmaf(v.w, f, y[3]);
        } else {
          const float2 v = *reinterpret_cast<const float2*>(src);
          y[0] = fmaf(v.x, f, y[0]);
          y[1] = fmaf(v.y, f, y[1]);
        }
      }
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
        p.lse[static_cast<int64_t>(h) * p.tq + t.q0 + tok] = all == 0.f ? -INFINITY : (top - Cfg<128, DV, F16>::kBias + log2f(all)) * kLn2;
      }
    }
  }
}

template <int DQK, int DV, bool F16>
cudaError_t launch(const PaParams& p, const void* tmap_k, const void* tmap_v, int ctas, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(pa_kernel<DQK, DV, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  if (!p.self_plan) {
    pa_plan_kernel<<<1, 1024, 0, stream>>>(p, ctas);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    count_launch();
  }
  e = launch_maybe_pdl(pa_kernel<DQK, DV, F16>, dim3(ctas), dim3(kThreads), kSmem, stream, !p.self_plan, p,
                       *reinterpret_cast<const CUtensorMap*>(tmap_k), *reinterpret_cast<const CUtensorMap*>(tmap_v));
  if (e != cudaSuccess) return e;
  count_launch();
  if (p.slots > 0) {
    e = launch_maybe_pdl(pa_merge_kernel<DV, F16>, dim3(ctas * 2), dim3(256), 0, stream, true, p);
    count_launch();
  }
  return e;
}

}  // namespace

cudaError_t launch_prompt_attention(const PaParams& p, int dqk, int dv, int dtype, const void* tmap_k, const void* tmap_v, int ctas,
                                    cudaStream_t stream) {
  const bool f16 = dtype == PTO_DT_F16;
  if (dqk == 64 && dv == 64) return f16 ? launch<64, 64, true>(p, tmap_k, tmap_v, ctas, stream) : launch<64, 64, false>(p, tmap_k, tmap_v, ctas, stream);
  if (dqk == 128 && dv == 128) return f16 ? launch<128, 128, true>(p, tmap_k, tmap_v, ctas, stream) : launch<128, 128, false>(p, tmap_k, tmap_v, ctas, stream);
  if (dqk == 192 && dv == 128) return f16 ? launch<192, 128, true>(p, tmap_k, tmap_v, ctas, stream) : launch<192, 128, false>(p, tmap_k, tmap_v, ctas, stream);
  return cudaErrorInvalidValue;
}

}  // namespace pto
