// serve.cu -- serving over long and shared KV caches: rotary positions per token (and into
// the cache), attention of a batch over a shared prefix and its own ragged caches, the
// attention weight each cache slot receives, and eviction by that weight.
//
// What the reference does in this place (server/src): one RoPE offset for the batch
// (model.cpp:588-606), a prefix cache that copies the prefix's K / V into every request's
// own cache (scheduler.cpp:121-168), caches bounded by max_context_len.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "fm_serve.cuh"

namespace fm {

// ------------------------------------------------------------------ rotary positions
// Pair i of a head turns by pos * turns[i] full turns; the product and its reduction to
// [-1/2, 1/2] are fp64 (at position 1e6 an fp32 product is off by 0.06 rad), the sine and
// cosine of the reduced turn fp32.  A CTA takes `tpb` tokens: their cos / sin are computed
// once into shared memory, then shared by all heads.  Bound: HBM, every element read and
// written once (16384 tokens of 36 heads of 128: 66 us out of cache, 4.6 TB/s; 57 us call after
// call).  Four items of a thread in flight before the angles took more registers and were slower
// (16% at that size).
constexpr int kRopeThreads = 256;

namespace {

FM_DEV void rotate(float x1, float x2, float2 cs, float& o1, float& o2) {
  o1 = x1 * cs.x - x2 * cs.y;
  o2 = x1 * cs.y + x2 * cs.x;
}

FM_DEV float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
FM_DEV float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// source and destination rows of head slot `hs` of token t; false: no destination
struct RopeRow {
  const uint16_t* src;
  uint16_t* dst;
  bool rot;
};

FM_DEV bool rope_row(const RopeBase& a, int64_t t, int hs, RopeRow& r) {
  if (hs < a.nq) {
    r.src = a.q + t * a.q_ld + static_cast<int64_t>(hs) * a.d;
    r.dst = a.q_out + t * a.qo_ld + static_cast<int64_t>(hs) * a.d;
    r.rot = true;
    return true;
  }
  const int slot = a.slots[t];
  if (slot < 0) return false;
  if (slot >= a.max_len) {
    if (hs == a.nq) report(a.err, DEVERR_BOUNDS);
    return false;
  }
  const int64_t b = t / a.L;
  hs -= a.nq;
  r.rot = hs < a.nkv;
  if (!r.rot) hs -= a.nkv;
  const int64_t row = ((b * a.nkv + hs) * a.max_len + slot) * a.d;
  r.src = (r.rot ? a.k : a.v) + t * a.kv_ld + static_cast<int64_t>(hs) * a.d;
  r.dst = (r.rot ? a.cache_k : a.cache_v) + row;
  return true;
}

}  // namespace

// VEC: the rotated part splits into whole 16-byte chunks (half: rotary / 2 a multiple of 8,
// traditional: rotary a multiple of 8); otherwise elements are taken pair by pair.
template <bool TRADITIONAL, bool VEC, int PAIRS>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeSet<PAIRS> a) {
  extern __shared__ float2 s_cs[];  // [tpb][rotary / 2]
  pdl_wait();
  pdl_trigger();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tpb;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.tpb), a.T - t0));
  const int half = a.rotary / 2;
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int tt = i / half, p = i - tt * half;
    double u = static_cast<double>(a.positions[t0 + tt]) * a.turns[p];
    u -= rint(u);
    float sn, cs;
    sincospif(static_cast<float>(2.0 * u), &sn, &cs);
    s_cs[i] = make_float2(cs * a.factor, sn * a.factor);
  }
  __syncthreads();
  const int slots = a.nq + 2 * a.nkv;
  const int d = a.d;
  if (VEC) {
    // items of a head: half layout: rotary / 16 chunk pairs; traditional: rotary / 8 chunks;
    // then the (d - rotary) / 8 chunks that are copied.  A v head takes the same items.
    const int rot_items = TRADITIONAL ? a.rotary / 8 : a.rotary / 16;
    const int items = rot_items + (d - a.rotary) / 8;
    const int total = nt * slots * items;
    for (int i = threadIdx.x; i < total; i += kRopeThreads) {
      const int it = i % items, hs_t = i / items;
      const int hs = hs_t % slots, tt = hs_t / slots;
      RopeRow r;
      if (!rope_row(a, t0 + tt, hs, r)) continue;
      const float2* cs = s_cs + tt * half;
      if (it >= rot_items) {
        const int c = a.rotary + 8 * (it - rot_items);
        *reinterpret_cast<uint4*>(r.dst + c) = *reinterpret_cast<const uint4*>(r.src + c);
        continue;
      }
      if (TRADITIONAL) {
        uint4 v = *reinterpret_cast<const uint4*>(r.src + 8 * it);
        if (r.rot) {
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float o1, o2;
            rotate(lo_f(w[e]), hi_f(w[e]), cs[4 * it + e], o1, o2);
            w[e] = pack_bf16x2(o1, o2);
          }
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(r.dst + 8 * it) = v;
      } else {
        uint4 v1 = *reinterpret_cast<const uint4*>(r.src + 8 * it);
        uint4 v2 = *reinterpret_cast<const uint4*>(r.src + half + 8 * it);
        if (r.rot) {
          uint32_t w1[4] = {v1.x, v1.y, v1.z, v1.w}, w2[4] = {v2.x, v2.y, v2.z, v2.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a1, a2, b1, b2;
            rotate(lo_f(w1[e]), lo_f(w2[e]), cs[8 * it + 2 * e], a1, a2);
            rotate(hi_f(w1[e]), hi_f(w2[e]), cs[8 * it + 2 * e + 1], b1, b2);
            w1[e] = pack_bf16x2(a1, b1);
            w2[e] = pack_bf16x2(a2, b2);
          }
          v1 = make_uint4(w1[0], w1[1], w1[2], w1[3]);
          v2 = make_uint4(w2[0], w2[1], w2[2], w2[3]);
        }
        *reinterpret_cast<uint4*>(r.dst + 8 * it) = v1;
        *reinterpret_cast<uint4*>(r.dst + half + 8 * it) = v2;
      }
    }
  } else {
    const int items = half + (d - a.rotary);
    const int total = nt * slots * items;
    for (int i = threadIdx.x; i < total; i += kRopeThreads) {
      const int it = i % items, hs_t = i / items;
      const int hs = hs_t % slots, tt = hs_t / slots;
      RopeRow r;
      if (!rope_row(a, t0 + tt, hs, r)) continue;
      if (it >= half) {
        const int c = a.rotary + it - half;
        r.dst[c] = r.src[c];
        continue;
      }
      const int e1 = TRADITIONAL ? 2 * it : it, e2 = TRADITIONAL ? 2 * it + 1 : it + half;
      const uint16_t h1 = r.src[e1], h2 = r.src[e2];
      if (r.rot) {
        float o1, o2;
        rotate(bf2f(h1), bf2f(h2), s_cs[tt * half + it], o1, o2);
        r.dst[e1] = f2bf(o1);
        r.dst[e2] = f2bf(o2);
      } else {
        r.dst[e1] = h1;
        r.dst[e2] = h2;
      }
    }
  }
}

template <int PAIRS>
static cudaError_t launch_rope_set(const RopeSet<PAIRS>& a, unsigned grid, cudaStream_t st) {
  const size_t smem = sizeof(float2) * a.tpb * (a.rotary / 2);
  const bool vec = a.traditional ? a.rotary % 8 == 0 : (a.rotary / 2) % 8 == 0;
  void (*kernel)(RopeSet<PAIRS>) = a.traditional ? (vec ? rope_kernel<true, true, PAIRS> : rope_kernel<true, false, PAIRS>)
                                                 : (vec ? rope_kernel<false, true, PAIRS> : rope_kernel<false, false, PAIRS>);
  return launch_pdl(kernel, grid, kRopeThreads, smem, st, a);
}

cudaError_t launch_rope(RopeArgs& a, int num_sms, cudaStream_t st) {
  // few tokens: one per CTA (latency); many: four share the cos / sin set-up's barrier
  a.tpb = a.T >= 8ll * num_sms ? 4 : 1;
  const unsigned grid = static_cast<unsigned>((a.T + a.tpb - 1) / a.tpb);
  if (a.rotary > kRopeMaxDim / 2) return launch_rope_set(a, grid, st);
  RopeSet<kRopeMaxDim / 4> b;
  static_cast<RopeBase&>(b) = a;
  std::memcpy(b.turns, a.turns, sizeof(b.turns));
  return launch_rope_set(b, grid, st);
}

// ------------------------------------------------------------------ attention, split over keys
// attn_split_kernel: a warp is a worker with a private ring of 16-key K / V tiles (cp.async,
// 16-byte chunks swizzled so that ldmatrix meets no bank twice), so nothing in the CTA waits
// for another warp.  S = Q K^T and O += P V are mma.sync m16n8k16: 16 query rows cost the tensor
// pipe next to nothing beside the loads.  Per tile and row the running maximum m and sum l in
// fp32, O rescaled by 2^(m_old - m_new).  Eight warps a SM with two tiles in flight each keep
// 128 KB under way.  Bound: HBM (16 sequences of 100-16001 slots, 4 kv heads of 128, 264 MB: 46 us,
// 5.8 TB/s, 88% of a copy).
namespace {

FM_DEV int seq_len(const CacheAttnArgs& a, int b) {
  const int n = a.split_own ? a.lens[b] : 0;
  return n < 0 || n > a.max_len ? 0 : n;  // reported by the merge
}

// tiles of one item of sequences [0, b), summed; whole warp, B <= a few thousand
FM_DEV int tiles_before(const CacheAttnArgs& a, int b) {
  const int lane = threadIdx.x & 31;
  int s = 0;
  for (int i = lane; i < b; i += 32) s += (seq_len(a, i) + kAttnTile - 1) / kAttnTile;
  return __reduce_add_sync(0xffffffffu, s);
}

FM_DEV int tiles_per_worker(const CacheAttnArgs& a, int total) {
  return max(kAttnMinTiles, (total + a.workers - 1) / a.workers);
}

FM_DEV void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

FM_DEV void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

// 16 bytes, or zeros when n is 0 (nothing is read then)
FM_DEV void cp_async16_or_zero(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

FM_DEV void lds128(uint32_t addr, uint4& v) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
}
FM_DEV void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
FM_DEV void lds32(uint32_t addr, uint32_t& v) {
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
}

}  // namespace

template <int D>
__global__ void __launch_bounds__(kAttnWarps * 32) attn_split_kernel(const CacheAttnArgs a) {
  constexpr int CH = D / 8;                          // 16-byte chunks of a row
  constexpr int KS = D / 16;                         // k-steps of Q K^T
  constexpr int NT = D / 8;                          // n-tiles of O
  constexpr uint32_t ROW = D * 2;                    // bytes of a row
  constexpr uint32_t TILE = kAttnTile * ROW;         // bytes of a K (or V) tile
  constexpr uint32_t STAGE = 2 * TILE;
  extern __shared__ __align__(128) uint8_t s_kv[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(s_kv) + warp * (kAttnStages * STAGE);
  const int worker = blockIdx.x * kAttnWarps + warp;
  if (!a.after_tc) pdl_wait();
  pdl_trigger();

  const int tp = (a.split_prefix + kAttnTile - 1) / kAttnTile;  // tiles of a prefix item
  const int np = a.nkv * a.rt_p, ns = a.nkv * a.rt_s;           // items of the prefix / of a sequence
  const int total_p = tp * np;
  const int total = total_p + ns * tiles_before(a, a.B);
  const int per = tiles_per_worker(a, total);
  int t = worker * per;
  const int t_end = min(total, t + per);
  if (t >= t_end) {
    if (a.after_tc) pdl_wait();
    return;
  }

  // the item of tile t: sequence (-1: the prefix), item of it, tile of the item
  int b = -1, item, tiles;
  int tile;
  if (t < total_p) {
    item = t / tp;
    tile = t - item * tp;
    tiles = tp;
  } else {
    int rest = t - total_p;
    b = 0;
    while (true) {  // 32 sequences at a time
      const int i = b + lane;
      const int mine = i < a.B ? ns * ((seq_len(a, i) + kAttnTile - 1) / kAttnTile) : 0;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, incl > rest);
      if (past) {  // the first sequence whose tiles reach beyond `rest`
        const int f = __ffs(past) - 1;
        rest -= __shfl_sync(0xffffffffu, incl - mine, f);
        b += f;
        break;
      }
      rest -= __shfl_sync(0xffffffffu, incl, 31);
      b += 32;
      if (b >= a.B) break;  // t < total makes this unreachable
    }
    tiles = (seq_len(a, b) + kAttnTile - 1) / kAttnTile;
    item = rest / tiles;
    tile = rest - item * tiles;
  }

  while (t < t_end) {
    const int cnt = min(tiles - tile, t_end - t);
    const bool pre = b < 0;
    const int rts = pre ? a.rt_p : a.rt_s;
    const int kvh = item / rts, row0 = (item - kvh * rts) * kAttnRowTile;
    const int rows = pre ? a.B * a.L * a.group : a.L * a.group;
    const int len = pre ? a.split_prefix : seq_len(a, b);
    const int64_t tok0 = pre ? 0 : static_cast<int64_t>(b) * a.L;
    const int64_t base = pre ? kvh * a.p_head : (static_cast<int64_t>(b) * a.nkv + kvh) * a.max_len * D;
    const uint16_t* kb = (pre ? a.pk : a.ck) + base;
    const uint16_t* vb = (pre ? a.pv : a.cv) + base;

    auto load = [&](int j) {  // tile + j of the item into stage j
      if (j < cnt) {
        const uint32_t sk = ring + (j % kAttnStages) * STAGE, sv = sk + TILE;
        const int key0 = (tile + j) * kAttnTile;
#pragma unroll
        for (int i = 0; i < kAttnTile * CH / 32; ++i) {
          const int e = i * 32 + lane, r = e / CH, ch = e % CH;
          const int key = key0 + r;
          const uint32_t off = r * ROW + ((ch ^ (r & 7)) << 4);
          const int64_t src = static_cast<int64_t>(min(key, len - 1)) * D + ch * 8;
          const int n = key < len ? 16 : 0;  // rows past the length count as zeros
          cp_async16_or_zero(sk + off, kb + src, n);
          cp_async16_or_zero(sv + off, vb + src, n);
        }
      }
      cp_async_commit();
    };
    __syncwarp();  // the previous item's last reads of the ring are done
#pragma unroll
    for (int j = 0; j < kAttnStages - 1; ++j) load(j);

    // Q fragments of rows row0 + g and row0 + g + 8 (zeros past the last row), and the last
    // slot each of them sees
    uint32_t qa[KS][4];
    int lim[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = row0 + g + 8 * hf;
      const bool on = r < rows;
      const int tk = on ? r / a.group : 0;
      lim[hf] = !on ? -1 : pre ? len - 1 : len - a.L + tk;
      const uint16_t* q = a.q + (tok0 + tk) * a.q_ld + static_cast<int64_t>(kvh * a.group + (on ? r - tk * a.group : 0)) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qa[ks][hf] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * ks + 2 * c) : 0u;
        qa[ks][hf + 2] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * ks + 2 * c + 8) : 0u;
      }
    }
    const int sees = pre ? len - 1 : max(len - a.L + row0 / a.group, -1);  // the last slot that every row sees
    float* srow[2];  // where this thread's rows' scores go
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = row0 + g + 8 * hf;
      srow[hf] = a.scores && r < rows ? a.scores + ((static_cast<int64_t>(b) * a.nkv + kvh) * rows + r) * a.score_ld : nullptr;
    }
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int j = 0; j < cnt; ++j) {
      load(j + kAttnStages - 1);
      cp_async_wait<kAttnStages - 1>();
      __syncwarp();
      const uint32_t sk = ring + (j % kAttnStages) * STAGE, sv = sk + TILE;
      const int mi = lane >> 3, rr = lane & 7;
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int r = (mi >> 1) * 8 + rr, ch = 2 * ks + (mi & 1);
        uint32_t b0, b1, b2, b3;
        ldsm_x4(sk + r * ROW + ((ch ^ (r & 7)) << 4), b0, b1, b2, b3);
        mma_bf16_16816(s[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
        mma_bf16_16816(s[1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b2, b3);
      }
      // scale, visibility, online softmax; rows g (hf 0) and g + 8 (hf 1)
      uint32_t pa[2][2];
      float al[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = (tile + j) * kAttnTile + 8 * n + 2 * c + e;
            float& v = s[n][2 * hf + e];
            v = key <= lim[hf] ? v * a.scale_log2 : -INFINITY;
            mx = fmaxf(mx, v);
          }
        if (srow[hf]) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int key = (tile + j) * kAttnTile + 8 * n + 2 * c;
            if (key + 1 < len) *reinterpret_cast<float2*>(srow[hf] + key) = make_float2(s[n][2 * hf], s[n][2 * hf + 1]);
            else if (key < len) srow[hf][key] = s[n][2 * hf];
          }
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[hf], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every term is 0
        al[hf] = exp2f(m[hf] - ref);
        m[hf] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = exp2f(s[n][2 * hf] - ref), p1 = exp2f(s[n][2 * hf + 1] - ref);
          sum += p0 + p1;
          // the tensor product's operand, one rounding to bf16: outputs are off by 0.0021 (root mean square)
          // where P in fp32 gives 0.0017, their own rounding; two bf16 parts would double the product
          pa[n][hf] = pack_bf16x2(p0, p1);
        }
        l[hf] = l[hf] * al[hf] + sum;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][0] *= al[0];
        o[n][1] *= al[0];
        o[n][2] *= al[1];
        o[n][3] *= al[1];
      }
      // Infinities and NaN of V in slots that some of the rows do not see: 0 times them is NaN, so
      // they become zeros and the rows that do see them get them added.
      if (min((tile + j + 1) * kAttnTile, len) - 1 > sees) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kAttnTile * CH / 32; ++i) {
          const int e = i * 32 + lane;
          uint4 x;
          lds128(sv + e * 16, x);
          bad |= (tile + j) * kAttnTile + e / CH > sees &&
                 (x.x != finite_or_zero(x.x) || x.y != finite_or_zero(x.y) || x.z != finite_or_zero(x.z) || x.w != finite_or_zero(x.w));
        }
        if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
          for (int r = 0; r < kAttnTile; ++r) {
            const int key = (tile + j) * kAttnTile + r;
            if (key <= sees) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t x;
              lds32(sv + r * ROW + ((n ^ (r & 7)) << 4) + 4 * c, x);
              if (key <= lim[0]) add_not_finite(x, o[n][0], o[n][1]);
              if (key <= lim[1]) add_not_finite(x, o[n][2], o[n][3]);
            }
          }
          __syncwarp();
#pragma unroll 1
          for (int e = lane; e < kAttnTile * CH; e += 32) {
            if ((tile + j) * kAttnTile + e / CH <= sees) continue;
            uint4 x;
            lds128(sv + e * 16, x);
            sts128(sv + e * 16, make_uint4(finite_or_zero(x.x), finite_or_zero(x.y), finite_or_zero(x.z), finite_or_zero(x.w)));
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const int r = (mi & 1) * 8 + rr, ch = n + (mi >> 1);
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(sv + r * ROW + ((ch ^ (r & 7)) << 4), b0, b1, b2, b3);
        mma_bf16_16816(o[n], pa[0][0], pa[0][1], pa[1][0], pa[1][1], b0, b1);
        mma_bf16_16816(o[n + 1], pa[0][0], pa[0][1], pa[1][0], pa[1][1], b2, b3);
      }
      __syncwarp();  // the next iteration's load overwrites a stage read one step ago
    }
    cp_async_wait<0>();

    const int64_t slot = worker + (pre ? item : np + static_cast<int64_t>(b) * ns + item);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
      if (row0 + g + 8 * hf < rows) {
        const int64_t pr = slot * kAttnRowTile + g + 8 * hf;
        float* po = a.part_o + pr * D;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          *reinterpret_cast<float2*>(po + 8 * n + 2 * c) = make_float2(o[n][2 * hf], o[n][2 * hf + 1]);
        if (c == 0) a.part_ml[pr] = make_float2(m[hf], l[hf]);
      }
    }
    t += cnt;
    if (t >= t_end) break;
    tile = 0;
    ++item;
    if (item >= (pre ? np : ns)) {
      ++b;
      item = 0;
      while (seq_len(a, b) == 0) ++b;  // tiles are left, so a sequence that has some follows
    }
    tiles = b < 0 ? tp : (seq_len(a, b) + kAttnTile - 1) / kAttnTile;
  }
  // this kernel is not complete before the one in front of it is, so the merge need wait for one
  if (a.after_tc) pdl_wait();
}

// Bound by latency: a few dependent loads and the pieces' 512 bytes a row (512 rows of ~20 pieces: 5 us,
// 2048 of ~22: 10 us).  Joins the pieces of output rows: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, zeros when
// nothing was seen; lse2 = M + log2(sum) for the slot weights.
namespace {

template <int D>
struct RowJoin {
  static constexpr int V = D / 32;  // columns of a lane
  float acc[V] = {};
  float M = -INFINITY, S = 0.f;

  // n pieces, piece i in row row0 + i * step of a part buffer
  FM_DEV void add(const float* part_o, const float2* part_ml, int64_t row0, int step, int n) {
    if (n <= 2) add_by<2>(part_o, part_ml, row0, step, n);
    else add_by<8>(part_o, part_ml, row0, step, n);
  }

  // U: pieces whose loads are in flight together
  template <int U>
  FM_DEV void add_by(const float* part_o, const float2* part_ml, int64_t row0, int step, int n) {
    for (int i0 = 0; i0 < n; i0 += U) {
      float2 ml[U];
      float v[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        load(part_o, part_ml, row0 + static_cast<int64_t>(min(i0 + u, n - 1)) * step, ml[u], v[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < n) join(ml[u], v[u]);
    }
  }

  FM_DEV void load(const float* part_o, const float2* part_ml, int64_t pr, float2& ml, float (&v)[V]) const {
    const float* po = part_o + pr * D + (threadIdx.x & 31) * V;
    ml = part_ml[pr];
    if (V == 4) {
      const float4 t4 = *reinterpret_cast<const float4*>(po);
      v[0] = t4.x; v[1] = t4.y; v[2 % V] = t4.z; v[3 % V] = t4.w;
    } else {
      const float2 t2 = *reinterpret_cast<const float2*>(po);
      v[0] = t2.x; v[1] = t2.y;
    }
  }

  FM_DEV void join(const float2& ml, const float (&v)[V]) {
    if (ml.y == 0.f) return;  // the piece's keys are all hidden from this row
    const float mn = fmaxf(M, ml.x);
    const float wa = exp2f(M - mn), wb = exp2f(ml.x - mn);
    M = mn;
    S = S * wa + ml.y * wb;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = acc[e] * wa + v[e] * wb;
  }

  // row r of (sequence b, kv head kvh)
  FM_DEV void store(const CacheAttnArgs& a, int b, int kvh, int r) const {
    const int lane = threadIdx.x & 31;
    const float inv = S == 0.f ? 0.f : 1.f / S;
    const int tk = r / a.group;
    uint16_t* out = a.out + ((static_cast<int64_t>(b) * a.L + tk) * a.nh + kvh * a.group + (r - tk * a.group)) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2)
      *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
    if (a.lse2 && lane == 0)
      a.lse2[(static_cast<int64_t>(b) * a.nkv + kvh) * a.L * a.group + r] = S == 0.f ? INFINITY : M + log2f(S);
  }
};

}  // namespace

// Every row of a (sequence, kv head): a block takes a.merge_rows of them, a warp every fourth -- or
// SHARED, one row, a warp every fourth of its pieces, when there are few rows in all.
template <int D, bool SHARED>
__global__ void __launch_bounds__(128) attn_merge_kernel(const CacheAttnArgs a, const TcAttnArgs tp, const TcAttnArgs ts) {
  const int warp = threadIdx.x >> 5;
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int rows = a.L * a.group, first_row = blockIdx.x * a.merge_rows;
  // the split kernel's cut
  const int tp16 = (a.split_prefix + kAttnTile - 1) / kAttnTile;
  const int np = a.nkv * a.rt_p, ns = a.nkv * a.rt_s;
  int per = 1, own_first = 0, own_tiles = 0;
  if (a.workers) {
    per = tiles_per_worker(a, tp16 * np + ns * tiles_before(a, a.B));
    own_tiles = (seq_len(a, b) + kAttnTile - 1) / kAttnTile;
    own_first = tp16 * np + ns * tiles_before(a, b) + kvh * a.rt_s * own_tiles;
  }
  // the tcgen05 kernel's cuts, in places
  constexpr int kCost = TcAttnArgs::kItemCost;
  int per_p = 1, tiles_p = 0, per_s = 1, first_s = 0, tiles_s = 0, flat_s = 0;
  if (tp.workers) {
    tiles_p = tp.tiles(0);
    per_p = tc_places_per_worker(tp, (tiles_p + kCost) * tp.rps * tp.nkv);
  }
  if (ts.workers) {
    flat_s = b * ts.rps + first_row / kTcRows;
    tiles_s = ts.tiles(flat_s);
    per_s = tc_places_per_worker(ts, tc_places_before(ts, ts.items()) * ts.nkv);
    first_s = tc_places_before(ts, flat_s) * ts.nkv + kvh * (tiles_s + kCost) + kCost;
  }
  pdl_wait();
  pdl_trigger();
  // (here, since with caches of no slots this kernel may be the call's first)
  if (a.lens && threadIdx.x == 0 && blockIdx.x == 0 && kvh == 0 && (a.lens[b] < 0 || a.lens[b] > a.max_len))
    report(a.err, DEVERR_BOUNDS);
  __shared__ __align__(16) float s_acc[SHARED ? 3 : 1][SHARED ? D : 4];
  __shared__ float2 s_ml[3];
  constexpr int kEvery = SHARED ? 4 : 1;
  const int one = SHARED ? warp : 0;
  for (int r = first_row + (SHARED ? 0 : warp); r < min(rows, first_row + a.merge_rows); r += 4) {
    RowJoin<D> row;
    auto add = [&](const float* part_o, const float2* part_ml, int64_t row0, int step, int n) {
      if (one < n) row.add(part_o, part_ml, row0 + static_cast<int64_t>(one) * step, kEvery * step, (n - one + kEvery - 1) / kEvery);
    };
    auto split_join = [&](int first, int tiles, int64_t item, int rr) {
      if (tiles <= 0) return;
      const int w0 = first / per, w1 = (first + tiles - 1) / per;
      add(a.part_o, a.part_ml, (w0 + item) * kAttnRowTile + rr, kAttnRowTile, w1 - w0 + 1);
    };
    auto tc_join = [&](const TcAttnArgs& t, int pw, int first, int tiles, int64_t item, int rr) {
      if (tiles <= 0) return;
      const int w0 = first / pw, w1 = (first + tiles - 1) / pw;
      add(t.part_o, t.part_ml, (w0 + item) * kTcRows + rr, kTcRows, w1 - w0 + 1);
    };
    const int rp = b * rows + r;  // the row among all sequences'
    if (tp16 > 0) {
      const int item = kvh * a.rt_p + rp / kAttnRowTile;
      split_join(item * tp16, tp16, item, rp % kAttnRowTile);
    }
    if (tiles_p > 0) {
      const int item = rp / kTcRows * tp.nkv + kvh;
      tc_join(tp, per_p, item * (tiles_p + kCost) + kCost, tiles_p, item, rp % kTcRows);
    }
    if (own_tiles > 0)
      split_join(own_first + r / kAttnRowTile * own_tiles, own_tiles,
                 np + static_cast<int64_t>(b) * ns + kvh * a.rt_s + r / kAttnRowTile, r % kAttnRowTile);
    if (tiles_s > 0) tc_join(ts, per_s, first_s, tiles_s, static_cast<int64_t>(flat_s) * ts.nkv + kvh, r % kTcRows);
    if (SHARED) {
      constexpr int V = RowJoin<D>::V;
      const int lane = threadIdx.x & 31;
      if (warp > 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) s_acc[warp - 1][lane * V + e] = row.acc[e];
        if (lane == 0) s_ml[warp - 1] = make_float2(row.M, row.S);
      }
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = s_acc[w][lane * V + e];
        row.join(s_ml[w], v);
      }
    }
    row.store(a, b, kvh, r);
  }
}

// With attn_tc_kernel's own caches as the only source, the rows of the items that a cut between
// two workers splits: block (w, y) takes the item over the cut before worker w + 1, if that is
// the first cut of the item.
template <int D>
__global__ void __launch_bounds__(128) attn_merge_cut_kernel(const CacheAttnArgs a, const TcAttnArgs ts) {
  constexpr int kCost = TcAttnArgs::kItemCost;
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < a.B; b += 128)
      if (a.lens[b] < 0 || a.lens[b] > a.max_len) report(a.err, DEVERR_BOUNDS);
  const int per = tc_places_per_worker(ts, tc_places_before(ts, ts.items()) * ts.nkv);
  const int place = (blockIdx.x + 1) * per;
  pdl_wait();
  pdl_trigger();
  int flat, kvh, at;
  if (!tc_locate(ts, place, flat, kvh, at)) return;
  const int first = place - at + kCost, tiles = ts.tiles(flat);
  if (first >= place || first / per != static_cast<int>(blockIdx.x)) return;
  const int w1 = (first + tiles - 1) / per, n = w1 - static_cast<int>(blockIdx.x) + 1;
  const int b = flat / ts.rps, row0 = (flat - b * ts.rps) * kTcRows;
  const int rows = min(a.L * a.group - row0, kTcRows);
  // the first worker's piece in its slot 2 w + 1, the next ones' in their slots 2 w
  const int64_t slot0 = (2 * static_cast<int64_t>(blockIdx.x) + 1) * kTcRows, slot1 = slot0 + kTcRows;
  constexpr int R = 4;  // rows of a warp at a time: their pieces' loads are in flight together
  for (int r = (blockIdx.y * 4 + (threadIdx.x >> 5)) * R; r < rows; r += 4 * R * gridDim.y) {
    RowJoin<D> row[R];
    if (n == 2) {  // nearly every cut
      float2 ml[R][2];
      float v[R][2][RowJoin<D>::V];
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) row[i].load(ts.part_o, ts.part_ml, (u ? slot1 : slot0) + min(r + i, rows - 1), ml[i][u], v[i][u]);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) row[i].join(ml[i][u], v[i][u]);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        row[i].add(ts.part_o, ts.part_ml, slot0 + min(r + i, rows - 1), kTcRows, 1);
        row[i].add(ts.part_o, ts.part_ml, slot1 + min(r + i, rows - 1), 2 * kTcRows, n - 1);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (r + i < rows) row[i].store(a, b, kvh, row0 + r + i);
  }
}

// ------------------------------------------------------------------ slot weights
// acc[b, kvh, j] += sum over the kv head's query rows of 2^(s_rj - lse2_r), from the scores that
// attn_split_kernel left: 4 bytes a row and slot, where K again would be 2 * head_dim a slot
// (16 sequences of up to 16001 slots, 32/4 heads of 128: 54 us recomputing the scores, 6 us so).
// Four neighbouring slots a thread.
__global__ void __launch_bounds__(256) slot_weight_kernel(const CacheAttnArgs a) {
  __shared__ float s_lse[kAttnRowTile];
  __shared__ int s_lim[kAttnRowTile];  // the last slot that the row sees (whose lse may be NaN)
  const int b = blockIdx.z, kvh = blockIdx.y;
  int len = a.lens[b];
  if (len < 0 || len > a.max_len) len = 0;  // reported by the merge
  pdl_wait();
  pdl_trigger();
  if (static_cast<int>(blockIdx.x) * 1024 >= len) return;
  const int rows = a.L * a.group;
  const int64_t head = static_cast<int64_t>(b) * a.nkv + kvh;
  if (threadIdx.x < rows) {
    s_lse[threadIdx.x] = a.lse2[head * rows + threadIdx.x];
    s_lim[threadIdx.x] = len - a.L + static_cast<int>(threadIdx.x) / a.group;
  }
  __syncthreads();
  const int j = blockIdx.x * 1024 + threadIdx.x * 4;
  if (j >= len) return;
  const float* sc = a.scores + head * rows * a.score_ld + j;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (min(static_cast<int>(blockIdx.x) * 1024 + 1023, len - 1) <= len - a.L) {  // every row sees the block's slots
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(sc + static_cast<int64_t>(r) * a.score_ld);
      const float lse = s_lse[r];
      sum.x += exp2f(v.x - lse);
      sum.y += exp2f(v.y - lse);
      sum.z += exp2f(v.z - lse);
      sum.w += exp2f(v.w - lse);
    }
  } else {
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(sc + static_cast<int64_t>(r) * a.score_ld);
      const float lse = s_lse[r];
      const int lim = s_lim[r];
      sum.x += j <= lim ? exp2f(v.x - lse) : 0.f;
      sum.y += j + 1 <= lim ? exp2f(v.y - lse) : 0.f;
      sum.z += j + 2 <= lim ? exp2f(v.z - lse) : 0.f;
      sum.w += j + 3 <= lim ? exp2f(v.w - lse) : 0.f;
    }
  }
  float* acc = a.acc + head * a.max_len + j;
  acc[0] += sum.x;
  if (j + 1 < len) acc[1] += sum.y;
  if (j + 2 < len) acc[2] += sum.z;
  if (j + 3 < len) acc[3] += sum.w;
}

// Adds the pieces of a key tile's weights, in the workers' order.
__global__ void __launch_bounds__(kTcKeys) slot_weight_sum_kernel(const TcWeightArgs a) {
  const int b = blockIdx.z, kvh = blockIdx.y, flat = b * a.key_tiles + blockIdx.x;
  const int tiles = a.tiles(flat);
  pdl_wait();
  pdl_trigger();
  if (tiles == 0) return;
  const int per = tc_places_per_worker(a, tc_places_before(a, a.items()) * a.nkv);
  const int first = tc_places_before(a, flat) * a.nkv + kvh * (tiles + TcWeightArgs::kItemCost) + TcWeightArgs::kItemCost;
  const int64_t item = static_cast<int64_t>(flat) * a.nkv + kvh;
  float sum = 0.f;
  for (int w = first / per; w <= (first + tiles - 1) / per; ++w) {
    const float* p = a.part + (w + item) * kTcWeightParts * kTcKeys + threadIdx.x;
    sum += (p[0] + p[kTcKeys]) + (p[2 * kTcKeys] + p[3 * kTcKeys]);
  }
  const int key = blockIdx.x * kTcKeys + threadIdx.x;
  if (key < a.lens[b]) a.acc[(static_cast<int64_t>(b) * a.nkv + kvh) * a.max_len + key] += sum;
}

template <int D>
static cudaError_t attn_opt_in() {
  return cudaFuncSetAttribute(attn_split_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_split_smem(D));
}

cudaError_t evict_init(EvictClusters* c);

cudaError_t serve_init(EvictClusters* c) {
  cudaError_t e = attn_opt_in<128>();
  if (e == cudaSuccess) e = attn_opt_in<64>();
  if (e == cudaSuccess) e = evict_init(c);
  return e == cudaSuccess ? attn_tc_init() : e;
}

template <int D>
static cudaError_t launch_cache_attn_d(const CacheAttnArgs& a, const TcAttnArgs& p, const TcMapsKV& mp,
                                       const TcAttnArgs& s, const TcMapsKV& ms, const TcWeightArgs& w, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (p.workers) e = launch_attn_tc(p, D, mp.k, mp.v, st);
  if (e == cudaSuccess && s.workers) e = launch_attn_tc(s, D, ms.k, ms.v, st);
  if (e == cudaSuccess && a.workers)
    e = launch_pdl(attn_split_kernel<D>, a.workers / kAttnWarps, kAttnWarps * 32, attn_split_smem(D), st, a);
  if (e != cudaSuccess) return e;
  if (s.workers && s.direct) {
    if (s.workers > 1) e = launch_pdl(attn_merge_cut_kernel<D>, dim3(s.workers - 1, 4), 128, 0, st, a, s);
  } else {
    const dim3 rows((a.L * a.group + a.merge_rows - 1) / a.merge_rows, a.nkv, a.B);
    e = launch_pdl(a.merge_rows == 1 ? attn_merge_kernel<D, true> : attn_merge_kernel<D, false>, rows, 128, 0, st, a, p, s);
  }
  if (e != cudaSuccess || !a.acc) return e;
  if (!w.workers) return launch_pdl(slot_weight_kernel, dim3((a.max_len + 1023) / 1024, a.nkv, a.B), 256, 0, st, a);
  e = launch_slot_weight_tc(w, D, ms.k, ms.q, st);
  return e == cudaSuccess ? launch_pdl(slot_weight_sum_kernel, dim3(w.key_tiles, a.nkv, a.B), kTcKeys, 0, st, w) : e;
}

cudaError_t launch_cache_attn(const CacheAttnArgs& a, const TcAttnArgs& p, const TcMapsKV& mp, const TcAttnArgs& s,
                              const TcMapsKV& ms, const TcWeightArgs& w, int d, cudaStream_t st) {
  return d == 128 ? launch_cache_attn_d<128>(a, p, mp, s, ms, w, st) : launch_cache_attn_d<64>(a, p, mp, s, ms, w, st);
}

// ------------------------------------------------------------------ eviction
// evict_select_kernel (a CTA or a cluster per sequence and kv head) finds the n = min(len, budget) slots
// that stay: a radix select over 32-bit keys (protected slots the largest, then the weight's
// order-preserving bits, NaN as -inf), 8 bits a pass, ties to the lower slot.  The keys are read
// once, into shared memory where they fit.  It leaves the list of rows that move as
// (destination, source) pairs, for evict_move_kernel or, when there can only be a few, for
// itself.  In place only the holes below n are filled, by the kept slots from n on, both in
// ascending order: sources >= n, destinations < n, so no move reads what another writes.
constexpr int kEvictThreads = 1024;
constexpr int kEvictSmemKeys = 40960;  // 160 KB
constexpr int kEvictCopies = 8;        // of the counts: a lane's own of eight, so that a warp whose keys are
                                       // alike does not add to one word 32 times
// Where no head can have more moves than this, the select kernel makes them itself.  In place, rows of
// 128, inputs out of cache, GPU time with two launches / one: 32 heads that move one row 12.9 / 10.9 us
// whatever the limit, that move as many as it allows 64: 15.0 / 13.7, 128: 15.9 / 15.4, 256: 16.5 / 18.6,
// 512: 18.6 / 24.4 (128 of 4 heads: 14.8 / 14.5, of 128 heads 18.8 / 16.9, of 512 heads 61.4 / 60.8).
constexpr int kEvictFused = 128;

namespace {

FM_DEV uint32_t order_bits(float v) {
  if (v != v) v = -INFINITY;
  if (v == 0.f) v = 0.f;  // -0 ranks as 0
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;  // [0x007fffff, 0xff800000]
}

// exclusive prefix of warp w's count and the total, from every warp's count; whole warp
FM_DEV int warps_before(const int* counts, int warp, int* total) {
  const int lane = threadIdx.x & 31;
  const int v = counts[lane];
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
  *total = __reduce_add_sync(0xffffffffu, v);
  return before;
}

FM_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
FM_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
FM_DEV uint32_t in_cta(const void* p, int rank) {  // the address of p in another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
FM_DEV int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
FM_DEV int4 ld_cluster4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// every CTA of the cluster's *p, after a cluster barrier: the sum of those before `rank`, and of all; whole warp
FM_DEV int ctas_before(const int* p, int rank, int ctas, int* total) {
  const int lane = threadIdx.x & 31;
  const int v = lane < ctas ? ld_cluster(in_cta(p, lane)) : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < rank ? v : 0);
  *total = __reduce_add_sync(0xffffffffu, v);
  return before;
}

// rows [0, cnt) of the list, `warps` warps together, warp `w` of them: K and V rows, weights, positions
FM_DEV void evict_rows(const EvictArgs& a, int64_t bh, const int32_t* list_dst, const int32_t* list_src, int cnt, int w,
                       int warps) {
  constexpr int R = 4, U = 4;  // rows of a warp at a time, loads in flight
  const int lane = threadIdx.x & 31;
  const int ch = a.d / 8;
  for (int i0 = w * R; i0 < cnt; i0 += warps * R) {
    const int n = min(R, cnt - i0), total = n * 2 * ch;
    for (int e0 = lane; e0 < total; e0 += 32 * U) {
      uint4 v[U];
      uint16_t* to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = e0 + 32 * u;
        if (e >= total) continue;
        const int row = e / (2 * ch), c = e - row * 2 * ch;
        const bool is_v = c >= ch;
        const int col = (is_v ? c - ch : c) * 8;
        v[u] = *reinterpret_cast<const uint4*>((is_v ? a.cache_v : a.cache_k) + (bh * a.max_len + list_src[i0 + row]) * a.d + col);
        to[u] = (is_v ? a.out_v : a.out_k) + (bh * a.out_max_len + list_dst[i0 + row]) * a.d + col;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (e0 + 32 * u < total) *reinterpret_cast<uint4*>(to[u]) = v[u];
    }
    if (lane < n) {
      const int dst = list_dst[i0 + lane], src = list_src[i0 + lane];
      a.out_acc[bh * a.out_max_len + dst] = a.acc[bh * a.max_len + src];
      if (a.out_positions)
        a.out_positions[bh * a.out_max_len + dst] = a.positions ? a.positions[bh * a.max_len + src] : src;
    }
  }
}

}  // namespace

template <bool CLUSTER>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t s_dyn[];  // a bit per slot that stays, then the keys when they fit
  __shared__ __align__(16) int s_hist[256 * kEvictCopies];
  __shared__ __align__(16) int s_cnt[CLUSTER ? 2 : 1][256];  // this CTA's counts, by the pass's parity: the next
                                                             // pass's barrier says that all have read them
  __shared__ int s_ex[4];                                    // newest, equal keys, holes, tail for the cluster
  uint32_t* s_kept = s_dyn;
  uint32_t* s_keys = s_dyn + a.words;
  __shared__ int s_w[3][32];
  __shared__ int s_pick[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ctas = CLUSTER ? a.ctas : 1, rank = CLUSTER ? static_cast<int>(cluster_rank()) : 0;
  const int64_t bh = blockIdx.x / ctas;
  const int b = static_cast<int>(bh / a.nkv);
  pdl_wait();
  pdl_trigger();
  int len = a.lens[b];
  if (len < 0 || len > a.max_len) {
    if (threadIdx.x == 0 && rank == 0) report(a.err, DEVERR_BOUNDS);
    len = 0;
  }
  const int n = min(len, a.budget);
  const float* acc = a.acc + bh * a.max_len;
  const int32_t* pos = a.positions ? a.positions + bh * a.max_len : nullptr;
  int32_t* list_dst = a.list + bh * 2 * a.budget;
  int32_t* list_src = list_dst + a.budget;
  if (threadIdx.x == 0 && rank == 0 && a.fused && bh % a.nkv == 0) a.out_lens[b] = n;
  if (n == len) {  // all stay
    if (!a.in_place)
      for (int i = rank * kEvictThreads + threadIdx.x; i < n; i += ctas * kEvictThreads) list_dst[i] = list_src[i] = i;
    if (threadIdx.x == 0 && rank == 0 && !a.fused) {
      a.counts[2 * bh] = a.in_place ? 0 : n;
      a.counts[2 * bh + 1] = n;
    }
    return;
  }
  // this CTA's slots [lo, hi): whole 32-slot words
  const int words = (len + 31) / 32, share = (words + ctas - 1) / ctas;
  const int first_word = min(words, rank * share), last_word = min(words, first_word + share);
  const int lo = 32 * first_word, hi = min(len, 32 * last_word);
  // the newest position held
  int newest = len - 1;
  if (pos) {
    int mx = INT32_MIN;
#pragma unroll 8
    for (int i = lo + threadIdx.x; i < hi; i += kEvictThreads) mx = max(mx, pos[i]);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) s_w[0][warp] = mx;
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, s_w[0][lane]);
    if (CLUSTER) {
      if (threadIdx.x == 0) s_ex[0] = newest;
      cluster_sync();
      newest = __reduce_max_sync(0xffffffffu, lane < ctas ? ld_cluster(in_cta(&s_ex[0], lane)) : INT32_MIN);
    }
  }
  // protected: below `sinks`, or one of the `recent` positions up to the newest
  const int64_t oldest = static_cast<int64_t>(newest) - a.recent + 1;
  const int guard = oldest < INT32_MIN ? INT32_MIN : static_cast<int>(min(oldest, static_cast<int64_t>(INT32_MAX)));
  const bool any = a.recent > 0;  // (oldest passes the newest when none is)
  auto make_key = [&](int i) -> uint32_t {
    const int p = pos ? pos[i] : i;
    return p < a.sinks || (any && p >= guard) ? 0xffffffffu : order_bits(acc[i]);
  };
  const bool kept_here = a.keys_in_smem;
  auto key_of = [&](int i) -> uint32_t { return kept_here ? s_keys[i - lo] : make_key(i); };
  // radix select: the n-th largest key and how many keys equal to it stay
  uint32_t prefix = 0;
  int want = n;  // of the keys that match the prefix so far
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256 * kEvictCopies / 4) reinterpret_cast<int4*>(s_hist)[threadIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (shift == 24) {
#pragma unroll 8
      for (int i = lo + threadIdx.x; i < hi; i += kEvictThreads) {
        const uint32_t k = make_key(i);
        if (kept_here) s_keys[i - lo] = k;
        atomicAdd(&s_hist[(k >> 24) * kEvictCopies + lane % kEvictCopies], 1);
      }
    } else {
#pragma unroll 4
      for (int i = lo + threadIdx.x; i < hi; i += kEvictThreads) {
        const uint32_t k = key_of(i);
        if ((k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&s_hist[((k >> shift) & 255u) * kEvictCopies + lane % kEvictCopies], 1);
      }
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      const int4 x = reinterpret_cast<const int4*>(s_hist)[2 * threadIdx.x], y = reinterpret_cast<const int4*>(s_hist)[2 * threadIdx.x + 1];
      s_cnt[CLUSTER ? shift >> 3 & 1 : 0][threadIdx.x] = ((x.x + x.y) + (x.z + x.w)) + ((y.x + y.y) + (y.z + y.w));
    }
    if (CLUSTER) cluster_sync();
    else __syncthreads();
    if (warp == 0) {  // the bins from the largest down; lane l: 255 - 8 l to 248 - 8 l
      const int* bins = &s_cnt[CLUSTER ? shift >> 3 & 1 : 0][248 - 8 * lane];
      int c[8] = {}, mine = 0;
      for (int r = 0; r < ctas; ++r) {
        const int4 x = CLUSTER ? ld_cluster4(in_cta(bins + 4, r)) : *reinterpret_cast<const int4*>(bins + 4);
        const int4 y = CLUSTER ? ld_cluster4(in_cta(bins, r)) : *reinterpret_cast<const int4*>(bins);
        c[0] += x.w, c[1] += x.z, c[2] += x.y, c[3] += x.x;
        c[4] += y.w, c[5] += y.z, c[6] += y.y, c[7] += y.x;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += c[i];
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      int left = want - (incl - mine);
      if (left > 0 && left <= mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (left > 0 && left <= c[i]) {
            s_pick[0] = 255 - 8 * lane - i;
            s_pick[1] = left;
          }
          left -= c[i];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_pick[0]) << shift;
    want = s_pick[1];
  }
  // `want` of the keys equal to `prefix` stay, the lowest slots first.  A warp takes a contiguous
  // range of 32-slot words: first the equal keys are counted, then a bit says which slots stay, and
  // the holes below n and the kept slots from n on are counted; then a lane lists a word's.
  const int per = (last_word - first_word + 31) / 32;
  const int w0 = min(last_word, first_word + warp * per), w1 = min(last_word, w0 + per);
  int eq = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = 32 * w + lane;
    eq += __popc(__ballot_sync(0xffffffffu, i < len && key_of(i) == prefix));
  }
  if (lane == 0) s_w[0][warp] = eq;
  __syncthreads();
  int all;
  eq = warps_before(s_w[0], warp, &all);
  if (CLUSTER) {
    if (threadIdx.x == 0) s_ex[1] = all;
    cluster_sync();
    eq += ctas_before(&s_ex[1], rank, ctas, &all);
  }
  const uint32_t below = (1u << lane) - 1;
  auto under_n = [&](int w) {  // the slots of word w below n
    const int c = n - 32 * w;
    return c >= 32 ? 0xffffffffu : c <= 0 ? 0u : (1u << c) - 1;
  };
  int hole = 0, tail = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = 32 * w + lane;
    const uint32_t k = i < len ? key_of(i) : 0u;
    const bool is_eq = i < len && k == prefix;
    const uint32_t eqs = __ballot_sync(0xffffffffu, is_eq);
    const uint32_t kept = __ballot_sync(0xffffffffu, i < len && (k > prefix || (is_eq && eq + __popc(eqs & below) < want)));
    eq += __popc(eqs);
    if (lane == 0) s_kept[w - first_word] = kept;
    hole += __popc(~kept & under_n(w));
    tail += __popc(kept & ~under_n(w));
  }
  if (lane == 0) {
    s_w[1][warp] = hole;
    s_w[2][warp] = tail;
  }
  __syncthreads();
  int holes;
  hole = warps_before(s_w[1], warp, &holes);
  tail = warps_before(s_w[2], warp, &all);
  if (CLUSTER) {
    if (threadIdx.x == 0) {
      s_ex[2] = holes;
      s_ex[3] = all;
    }
    cluster_sync();
    hole += ctas_before(&s_ex[2], rank, ctas, &holes);
    tail += ctas_before(&s_ex[3], rank, ctas, &all);
  }
  for (int base = w0; base < w1; base += 32) {
    const int w = base + lane;
    const uint32_t kept = w < w1 ? s_kept[w - first_word] : 0u, under = w < w1 ? under_n(w) : 0u;
    uint32_t hm = ~kept & under, tm = kept & ~under, stay = a.in_place ? 0u : kept & under;
    int hi = __popc(hm), ti = __popc(tm);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int hu = __shfl_up_sync(0xffffffffu, hi, o), tu = __shfl_up_sync(0xffffffffu, ti, o);
      if (lane >= o) {
        hi += hu;
        ti += tu;
      }
    }
    int at = hole + hi - __popc(hm);
    // copied elsewhere, the slots that keep their places follow the moves
    int to = holes + 32 * w - at;
    for (; hm; hm &= hm - 1) list_dst[at++] = 32 * w + __ffs(hm) - 1;
    at = tail + ti - __popc(tm);
    for (; tm; tm &= tm - 1) list_src[at++] = 32 * w + __ffs(tm) - 1;
    for (; stay; stay &= stay - 1, ++to) list_dst[to] = list_src[to] = 32 * w + __ffs(stay) - 1;
    hole += __shfl_sync(0xffffffffu, hi, 31);
    tail += __shfl_sync(0xffffffffu, ti, 31);
  }
  // (a CTA leaves after the others' last reads of its shared memory)
  if (CLUSTER) cluster_sync();
  if (a.fused) {
    if (!CLUSTER) __syncthreads();  // the lists are written (and read by this block or cluster alone)
    evict_rows(a, bh, list_dst, list_src, holes, rank * 32 + warp, ctas * 32);
  } else if (threadIdx.x == 0 && rank == 0) {
    a.counts[2 * bh] = a.in_place ? holes : n;
    a.counts[2 * bh + 1] = n;
  }
}

__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a) {
  const int64_t bh = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int cnt = a.counts[2 * bh];
  if (blockIdx.x == 0 && threadIdx.x == 0 && bh % a.nkv == 0) a.out_lens[bh / a.nkv] = a.counts[2 * bh + 1];
  const int32_t* list_dst = a.list + bh * 2 * a.budget;
  evict_rows(a, bh, list_dst, list_dst + a.budget, cnt, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8);
}

cudaError_t evict_init(EvictClusters* c) {
  const int smem = kEvictSmemKeys * 4 + kEvictSmemKeys / 8;
  cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  for (int ctas : {2, 4}) {
    cudaLaunchConfig_t l = {};
    l.gridDim = dim3(ctas);
    l.blockDim = dim3(kEvictThreads);
    l.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
    l.attrs = &attr;
    l.numAttrs = 1;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(ctas == 2 ? &c->twos : &c->fours, evict_select_kernel<true>, &l);
  }
  return e;
}

cudaError_t launch_evict(EvictArgs a, bool lens_apart, const EvictClusters& clusters, int num_sms, cudaStream_t st) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.nkv;
  const int64_t most = a.in_place ? std::min(a.budget, std::max(0, a.max_len - a.budget)) : a.budget;
  a.ctas = evict_ctas(heads, a.max_len, clusters);
  a.words = ((a.max_len + 31) / 32 + a.ctas - 1) / a.ctas;
  a.keys_in_smem = a.words * 32 <= kEvictSmemKeys;
  // a step that is a few slots over: no second launch (unless out_lens is lens, which other blocks
  // of the sequence may not have read yet)
  a.fused = a.in_place && most <= kEvictFused && lens_apart;
  const cudaError_t e = launch_pdl_cluster(a.ctas > 1 ? evict_select_kernel<true> : evict_select_kernel<false>, a.ctas,
                                           static_cast<unsigned>(heads * a.ctas), kEvictThreads,
                                           a.words * 4 * (a.keys_in_smem ? 33 : 1), st, a);
  if (e != cudaSuccess || a.fused) return e;
  const int64_t want = std::max<int64_t>(1, (num_sms * 8 + heads - 1) / heads);
  const unsigned gx = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((most + 31) / 32, want)));
  return launch_pdl(evict_move_kernel, dim3(gx, static_cast<unsigned>(heads)), 256, 0, st, a);
}

}  // namespace fm
