// Parameters of the prompt attention (prompt_attention.cu) and the sizes its workspace is counted with.
#pragma once
#include "common.cuh"

namespace pto {

constexpr int kPaRows = 256;        // query rows (tokens x heads of a group) of a work item: two MMA tiles
constexpr int kPaKeys = 128;        // keys of a tile
constexpr int kPaSmallTiles = 256;  // tables of up to this many row tiles are built by every CTA for itself
constexpr int kPaMinPiece = 4;      // key tiles that a piece of an item has at least
constexpr int kPaCtas = 148;        // at most
constexpr int kPaSlots = 8 * kPaCtas;  // pieces of items that are in pieces, at most

// A row tile of a sequence. Its pieces are numbers [piece, piece + pieces) of every head; those of a tile in several pieces have
// slots [slot, slot + pieces) x heads of the partial results.
struct alignas(16) PaTile {
  int q0, lq, k0, lk;  // first token and tokens, first key and keys of its sequence
  int row0, pieces, piece, slot;
};
struct PaHead {
  int tiles, pieces;  // of the table
  int next;           // items handed out beyond the first ones
  int cut;            // tiles up to the last one that is in several pieces
};

struct PaParams {
  const void* q;
  void* out;
  const void* v;   // (values that are not finite are looked up once more)
  float* lse;      // [hq, tq] or null
  int64_t q_token, q_head, out_token, out_head, v_token, v_head;
  const int32_t *cu_q, *cu_k;
  int tq, tk, b, hq, hkv, group;
  uint32_t group_mul;  // row / group = row * group_mul >> group_shift
  int group_shift;
  int out_wide;  // rows of the output on 32-byte boundaries
  int q_map;  // query tiles are boxes of a tensor map (the group divides 128)
  int causal, head_set;  // head_set: key heads that are worked on together (what L2 holds)
  float scale, scale_log2;
  int max_tiles, slot_rows;
  int self_plan;        // every CTA builds the table
  uint8_t* tables;      // PaHead, PaTile [max_tiles], int first [b + 1]; `table_stride` bytes a CTA
  int64_t table_stride;
  float2* part_ml;      // [slot][slot_rows]: maximum of the scores, sum
  float* part_o;        // [slot][slot_rows][dv]
  int slots;            // 0: no item can be in pieces
  int32_t* status;
};

cudaError_t launch_prompt_attention(const PaParams& p, int dqk, int dv, int dtype, const void* tmap_q, const void* tmap_k,
                                    const void* tmap_v, int ctas, cudaStream_t stream);

}  // namespace pto
