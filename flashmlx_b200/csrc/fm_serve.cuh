// fm_serve.cuh -- arguments of the serving kernels (serve.cu).
#pragma once

#include "fm_internal.cuh"

namespace fm {

constexpr int kRopeMaxDim = 256;  // largest head size of the rotary kernels

struct RopeArgs {
  const uint16_t* q;        // [T, q_ld]: nq heads of d
  uint16_t* q_out;          // [T, qo_ld]
  int64_t q_ld, qo_ld;
  const uint16_t* k;        // append: [T, kv_ld]: nkv heads of d, rotated into cache_k
  const uint16_t* v;        // append: copied into cache_v
  int64_t kv_ld;
  uint16_t* cache_k;        // [B, nkv, max_len, d]
  uint16_t* cache_v;
  const int32_t* positions; // [T]
  const int32_t* slots;     // [T] cache slot of token t of sequence t / L; < 0: not written
  int64_t T;
  int nq, nkv, d, rotary, L, max_len, traditional;
  int tpb;                  // tokens of a CTA
  float factor;             // on cos and sin
  uint32_t* err;
  double turns[kRopeMaxDim / 2];  // full turns per position of each pair
};

constexpr int kAttnTile = 16;        // keys of a tile
constexpr int kAttnRowTile = 16;     // query rows of an item
constexpr int kAttnMinTiles = 4;     // least tiles of a worker's range
constexpr int kAttnWarps = 4;        // workers of a CTA
constexpr int kAttnBlocksPerSm = 2;
constexpr int kAttnStages = 3;       // ring of K / V tiles of a worker
constexpr int attn_split_smem(int d) { return kAttnWarps * kAttnStages * 2 * kAttnTile * d * 2; }

struct CacheAttnArgs {
  const uint16_t* q;        // [B * L, q_ld]: nh heads of d
  int64_t q_ld;
  const uint16_t* pk;       // [nkv, p_head / d, d] shared prefix
  const uint16_t* pv;
  int64_t p_head;           // elements from one prefix head to the next
  const uint16_t* ck;       // [B, nkv, max_len, d] the sequences' own caches
  const uint16_t* cv;
  const int32_t* lens;      // [B] or null: no own caches
  uint16_t* out;            // [B * L, nh * d]
  float* acc;               // [B, nkv, max_len] or null
  int B, L, nh, nkv, group, max_len, prefix_len;
  float scale_log2;         // softmax scale * log2(e)
  int rt_p, rt_s;           // row tiles of the prefix items / of a sequence's items, per kv head
  int workers;
  float* part_o;            // [slots][16][d]
  float2* part_ml;          // [slots][16] (maximum in log2 units, sum)
  float* lse2;              // [B * L, nh] or null
  uint32_t* err;
};

struct CacheAttnPlan {
  int64_t rt_p = 0, rt_s = 0;
  int workers = 0;
  size_t off_ml = 0, off_lse = 0, bytes = 0;
};
CacheAttnPlan cache_attn_plan(int B, int L, int nh, int nkv, int d, int prefix_len, bool scored, int num_sms);

struct EvictArgs {
  const uint16_t* cache_k;  // [B, nkv, max_len, d]
  const uint16_t* cache_v;
  const float* acc;         // [B, nkv, max_len]
  const int32_t* positions; // [B, nkv, max_len] or null: a slot's position is its index
  const int32_t* lens;      // [B]
  uint16_t* out_k;          // [B, nkv, out_max_len, d]; cache_k when in place
  uint16_t* out_v;
  float* out_acc;
  int32_t* out_positions;   // or null
  int32_t* out_lens;        // [B]
  int B, nkv, d, max_len, out_max_len, budget, sinks, recent;
  int in_place;
  int32_t* list;            // [B * nkv][2][budget] destinations, sources
  int32_t* counts;          // [B * nkv][2] rows to move, slots that stay
  uint32_t* err;
};

cudaError_t launch_rope(RopeArgs a, int num_sms, cudaStream_t st);
cudaError_t cache_attn_init();
cudaError_t launch_cache_attn(const CacheAttnArgs& a, int d, cudaStream_t st);
cudaError_t launch_evict(const EvictArgs& a, int num_sms, cudaStream_t st);

}  // namespace fm
