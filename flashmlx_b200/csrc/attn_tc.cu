// attn_tc.cu -- attention of many query rows over a key range on tcgen05 (sm_100a): the shared
// prefix of a batch, and the new tokens' rows of a sequence when they are more than a warp's
// tile.  fm_serve.cuh describes the order of the work and its split over workers.
//
// A worker is a CTA, one per SM.  An item is a kv head's keys and up to 256 query rows (the
// group's heads of neighbouring tokens, so that every head that shares the keys shares the
// loads), two 128-row tiles.  Two streams of 128 softmax threads, a row each, share the tensor
// pipe and every K / V tile: with more than 128 rows a stream has its own row tile and all keys,
// with fewer both have the same rows and a stream takes half of each tile's keys; their halves
// are joined in shared memory when the piece ends.
//
//   warps 0-3, 4-7  stream 0, 1: Q rows to shared memory (the next piece's come in while a
//                   piece's last product runs, and are stored before its O leaves, so that the
//                   next S are computed meanwhile); per 64 keys S out of TMEM, scale and
//                   visibility, online softmax, P back into TMEM over S (bf16 pairs); at the
//                   end O out of TMEM, through shared memory so that the stores are whole lines
//   warps 8, 9      MMA issuers of streams 0 and 1: S = Q K^T (both operands K-major in shared
//                   memory) and O += P V (P in TMEM, V as loaded: keys x head, i.e. MN-major).
//                   One each, since an issuer's own waits and commits took ~950 cycles a step
//                   where the products take 640
//   warp 10         TMA loads of K / V tiles of 128 keys into a ring (four tiles of 128 columns:
//                   a fifth would take the room of the stage that O leaves through)
//
// TMEM: per stream two S / P buffers of 64 columns and head_dim columns of O.  A step is 64 keys
// of a stream; S of step n + 2 is issued right after P V of step n, into the buffer that step
// n's P leaves, so S of step n + 1 is there before the stream is done with step n and the streams
// never wait for the pipe's latency.  (With one S of 128 keys a stream -- all that fits next to
// O -- the chain S, softmax, P V, S took 3950 cycles a tile where the products take 2048.)
//
// P is 2^(s - ref) with a row's ref the maximum of its first step, moved (and O rescaled, by the
// stream itself) only when a later term passes it by more than 8: O in TMEM is rarely touched,
// and P stays below 2^8 and keeps its relative precision.
//
// Bound: the exponentials of the two streams, which fall into step (64 keys: ~1200 of 1700 cycles
// with both at the special-function units, 1063 at their rate).  A prompt of 4096 tokens, 32/4 heads of
// 128: 146 us, 0.94 PFLOP/s; 64 sequences' rows over 32768 shared keys: 45 us, of which a worker has 11,000
// cycles before its first S (3200 launch and cut, 3900 Q, 3900 S), 30 steps of ~1750, 8500 for O.
#include "fm_serve.cuh"

namespace fm {
namespace {

constexpr int kThreads = 352;
constexpr int kMmaWarp = 8;      // and 9; warp 10 loads
constexpr int kStep = 64;        // keys of a stream's step

template <int D>
struct Shape {
  static constexpr int kHalf = D / 64;                       // 64-column halves of a row
  static constexpr uint32_t kTileBytes = kTcKeys * D * 2;    // a K, V or 128-row Q tile
  static constexpr int kSlots = D == 128 ? 4 : 8;            // ring of K / V tiles
  static constexpr uint32_t kStage = 32 * 128;               // a warp's: 32 rows of 128 bytes
  static constexpr uint32_t kSmem = 1024 + (2 + kSlots) * kTileBytes + kMmaWarp * kStage;
};

struct Bars {
  uint64_t qfull[2], sfull[2][2], pfull[2][2], ofull, tail, done[2], otail[2];
  uint64_t kvfull[8], kvempty[8], half[4];
  uint32_t tmem;
  int abort_flag;
  uint32_t hidden[8];  // [i % 8] == i + 1: of the CTA's piece i, values were set to zero (the loader is
                       // at most four pieces ahead: the ring holds eight tiles)
};

FM_DEV void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}

// descriptor of a [K rows x 64 N columns] tile in the 128-byte swizzle read as the N x K operand
// (MN-major): 8 K rows 1024 B apart, the next 64 columns `cols` bytes on
FM_DEV uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t cols) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(cols >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

FM_DEV float ex2(float x) {  // 2^x, 2 ulp; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

FM_DEV void tma_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// 32 columns of this lane's row, without waiting for them
FM_DEV void tmem_ld32_async(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
FM_DEV void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
FM_DEV void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
FM_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// bounded wait that ignores the abort flag: drains copies and products in flight
FM_DEV bool wait_drained(uint64_t* bar, uint32_t parity, uint32_t* err) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - t0 > kWaitBudgetCycles) {
      report(err, DEVERR_TIMEOUT);
      return false;
    }
  }
  return true;
}

}  // namespace

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ TcAttnArgs a,
                                                             const __grid_constant__ CUtensorMap map_k,
                                                             const __grid_constant__ CUtensorMap map_v) {
  using S = Shape<D>;
  constexpr int NS = S::kSlots;
  extern __shared__ uint8_t s_raw[];
  __shared__ Bars bars;
  // tiles on 1024-byte boundaries, as the swizzle's pattern needs
  const uint32_t pad = (1024u - (smem_u32(s_raw) & 1023u)) & 1023u;
  uint8_t* s_q = s_raw + pad;                        // [2][kTileBytes]
  uint8_t* s_kv = s_q + 2 * S::kTileBytes;           // [NS][kTileBytes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars.abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.qfull[i], 4);  // a warp's arrival each
      for (int j = 0; j < 2; ++j) {
        mbar_init(&bars.sfull[i][j], 1);
        mbar_init(&bars.pfull[i][j], 4);
      }
    }
    mbar_init(&bars.ofull, 2);
    mbar_init(&bars.tail, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.done[i], 1);
      mbar_init(&bars.otail[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bars.half[i], 2);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.kvfull[i], 1);
      mbar_init(&bars.kvempty[i], 2);
    }
    bars.abort_flag = 0;
    for (int i = 0; i < 8; ++i) bars.hidden[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  pdl_wait();
  pdl_trigger();
  const int per = tc_places_per_worker(a, tc_places_before(a, a.items()) * a.nkv);

  TcPiece it;
  tc_first(a, blockIdx.x, per, it);
  const int rows = a.L * a.group;

  if (warp < kMmaWarp) {
    // ---------------------------------------------------------------- softmax streams
    const int s = warp >> 2;
    const int quad = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + lanes + s * kTcKeys, t_o = tmem + lanes + 2 * kTcKeys + s * D;
    uint8_t* q_tile = s_q + s * S::kTileBytes;
    uint8_t* stage = s_kv + NS * S::kTileBytes + warp * S::kStage;
    constexpr int CPR = D / 8, RPI = 32 / CPR;  // 16-byte chunks of a row, rows a warp brings at once
    uint4 qv[32 / RPI];
    // ---- Q: stream s brings tile s (with one tile of rows stream 0 alone)
    auto fetch_q = [&](const TcPiece& p) {
      const int b = a.by_rps.divide(p.flat), row_base = (p.flat - b * a.rps) * kTcRows;
      const bool mine = p.cnt > 0 && (s == 0 || rows - row_base > kTcKeys);
      const uint16_t* q = a.q + static_cast<int64_t>(b) * a.L * a.q_ld + static_cast<int64_t>(p.kvh) * a.group * D + lane % CPR * 8;
      const int r0 = row_base + s * kTcKeys + quad * 32 + lane / CPR;
#pragma unroll
      for (int i = 0; i < 32 / RPI; ++i) {
        const int r = r0 + i * RPI, tk = a.by_group.divide(r);
        qv[i] = make_uint4(0, 0, 0, 0);
        if (mine && r < rows) qv[i] = *reinterpret_cast<const uint4*>(q + tk * a.q_ld + (r - tk * a.group) * D);
      }
    };
    // both streams arrive for every piece, so that neither falls behind by a phase of `ofull`
    auto store_q = [&](const TcPiece& p) {
      if (p.cnt <= 0) return;
      if (s == 0 || rows - (p.flat - a.by_rps.divide(p.flat) * a.rps) * kTcRows > kTcKeys) {
        const int ch = lane % CPR;
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
          uint4 v = qv[i];
          v.x ^= a.q_sign;  // a negative scale is taken as its size, with -q
          v.y ^= a.q_sign;
          v.z ^= a.q_sign;
          v.w ^= a.q_sign;
          *reinterpret_cast<uint4*>(q_tile + (ch >> 3) * (kTcKeys * 128) +
                                    sw128_off(quad * 32 + i * RPI + lane / CPR, ch & 7)) = v;
        }
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.qfull[s]);
    };
    uint32_t g = 0;  // steps of this stream: step g is in buffer g % 2
    int oph = 0, half_ph = 0, tails = 0;
    bool ok = true;
    // the two streams' warps of the same rows see what the other wrote
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.half[quad]);
      const bool got = __all_sync(0xffffffffu, mbar_wait(&bars.half[quad], half_ph & 1, abort_flag, a.err));
      ++half_ph;
      return got;
    };
    fetch_q(it);
    store_q(it);
    while (it.cnt > 0) {
      const int b = a.by_rps.divide(it.flat), row_base = (it.flat - b * a.rps) * kTcRows;
      const bool pair = rows - row_base > kTcKeys;
      const int len = tc_len(a, b);
      const int64_t tok0 = static_cast<int64_t>(b) * a.L;
      const int rl = quad * 32 + lane;
      const int r = row_base + (pair ? s * kTcKeys : 0) + rl;
      const bool on = r < rows;
      const int tk = on ? a.by_group.divide(r) : 0;
      const int lim = !on ? -1 : a.causal ? len - a.L + tk : len - 1;  // the last key this row sees
      const bool live = row_base + (pair ? s * kTcKeys : 0) + quad * 32 < rows;
      const int steps = pair ? 2 * it.cnt : it.cnt;
      float ref = -INFINITY, l = 0.f;
      int key0 = it.tile * kTcKeys + (pair ? 0 : s * kStep);
#pragma unroll 1
      for (int n = 0; n < steps; ++n, ++g, key0 += pair ? kStep : kTcKeys) {
        const uint32_t buf = g & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.sfull[s][buf], g >> 1 & 1, abort_flag, a.err))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (live) {
          const uint32_t t_b = t_s + buf * kStep;
          float v[kStep];
#pragma unroll
          for (int c = 0; c < kStep; c += 32) tmem_ld32_async(t_b + c, v + c);
          tmem_wait_ld();
          if (__any_sync(0xffffffffu, lim < key0 + kStep - 1)) {
#pragma unroll
            for (int c = 0; c < kStep; ++c) v[c] = key0 + c <= lim ? v[c] : -INFINITY;
          }
          auto maximum = [&]() {
            float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int c = 4; c < kStep; ++c) m4[c & 3] = fmaxf(m4[c & 3], v[c]);
            return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
          };
          float sum;
          auto exponentials = [&]() {
            const float base = ref == -INFINITY ? 0.f : -ref;
            float sum4[4] = {0.f, 0.f, 0.f, 0.f};
            uint4 w[8];
            uint32_t* pw = reinterpret_cast<uint32_t*>(w);
#pragma unroll
            for (int c = 0; c < kStep / 2; ++c) {
              const float p0 = ex2(fmaf(v[2 * c], a.scale_log2, base)), p1 = ex2(fmaf(v[2 * c + 1], a.scale_log2, base));
              sum4[2 * c & 3] += p0;
              sum4[2 * c + 1 & 3] += p1;
              // the tensor product's operand, one rounding to bf16: outputs are off by 0.0023 (root mean
              // square) where P in fp32 gives 0.0017, their own rounding; two parts would double P V
              pw[c] = pack_bf16x2(p0, p1);
            }
            tmem_st32(t_b, w);
            sum = (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
          };
          // ref is the maximum of the first step that a row sees anything in.  Later a row's sum says
          // whether ref still serves: a term above 2^8 makes it larger than 2^8 (many smaller terms may
          // too, which costs an unneeded move).  That saves the maximum, as long a job as the
          // exponentials are; in the rare case that ref moves the step's exponentials are done again.
          bool fresh = ref == -INFINITY && lim >= key0;
          if (!__any_sync(0xffffffffu, fresh)) {
            exponentials();
            fresh = sum > 256.f;
          }
          if (__any_sync(0xffffffffu, fresh)) {
            const float nref = fresh ? fmaxf(maximum(), ref) : ref;
            const float f = ref == -INFINITY ? 0.f : ex2(ref - nref);
            if (n > 0 && __any_sync(0xffffffffu, f != 1.f)) {
              // The product of step n - 1, which writes O, has to be complete: S of step n + 1 was
              // issued right after it (S of this step only after that of step n - 2).  At the last
              // step there is none, and `otail` says so.
              uint64_t* bar = n + 1 < steps ? &bars.sfull[s][buf ^ 1] : &bars.otail[s];
              const uint32_t ph = n + 1 < steps ? (g + 1) >> 1 & 1 : tails & 1;
              if (!__all_sync(0xffffffffu, mbar_wait(bar, ph, abort_flag, a.err))) {
                ok = false;
                break;
              }
              tc_fence_after();
              l *= f;
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                tmem_ld16(t_o + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f;
                tmem_st16(t_o + c, o);
              }
            }
            ref = nref;
            exponentials();
          }
          l += sum;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pfull[s][buf]);
      }
      tails += steps > 1;
      TcPiece nx = it;
      tc_next(a, nx);
      fetch_q(nx);
      if (!ok || !__all_sync(0xffffffffu, mbar_wait(&bars.ofull, oph & 1, abort_flag, a.err))) {
        ok = false;
        break;
      }
      const bool spoiled = *const_cast<const volatile uint32_t*>(&bars.hidden[oph & 7]) == static_cast<uint32_t>(oph) + 1;
      ++oph;
      tc_fence_after();
      store_q(nx);  // S of the next piece's first steps while this one's O leaves
      const bool whole = a.direct && it.cnt == it.tiles;
      if (live) {
        const int64_t row = (tok0 + tk) * a.nh + it.kvh * a.group + (r - tk * a.group);
        const int64_t pr = tc_slot(a, blockIdx.x, it) * kTcRows + (pair ? s * kTcKeys : 0) + quad * 32;
        const uint32_t on_rows = __ballot_sync(0xffffffffu, on);
        const int rsub = lane >> 3, csub = lane & 7;
        float fac = 1.f;  // on this stream's O
        if (!pair) {      // one reference for both streams' halves
          const int other = s == 0 ? 4 * static_cast<int>(S::kStage) : -4 * static_cast<int>(S::kStage);
          reinterpret_cast<float2*>(stage)[lane] = make_float2(ref, l);
          ok = meet();
          const volatile float* theirs = reinterpret_cast<const volatile float*>(stage + other) + 2 * lane;
          const float2 o = make_float2(theirs[0], theirs[1]);
          ok = ok && meet();
          if (!ok) break;
          const float top = fmaxf(ref, o.x);
          fac = ref == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(ref - top);
          l = l * fac + (o.x == -INFINITY ? o.y : o.y * ex2(o.x - top));
          ref = top;
        }
        const float mul = whole ? (l == 0.f ? 0.f : fac / l) : fac;
        // a 128-byte line of each row at a time: 32 fp32 or 64 bf16 columns
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          __syncwarp();
          tmem_ld32(t_o + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= mul;
          if (!pair) {  // stream 1 hands its half over
            if (s == 1) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(stage + sw128_off(lane, e)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            if (!meet()) {
              ok = false;
              break;
            }
            if (s == 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 h = *reinterpret_cast<const float4*>(stage + 4 * S::kStage + sw128_off(lane, e));
                o[4 * e] += h.x;
                o[4 * e + 1] += h.y;
                o[4 * e + 2] += h.z;
                o[4 * e + 3] += h.w;
              }
            }
            if (!meet()) {
              ok = false;
              break;
            }
            if (s == 1) continue;
          }
          if (spoiled) {  // the values that the loader took out, for the rows that see them
            const uint16_t* vr = a.v + (static_cast<int64_t>(b) * a.nkv + it.kvh) * a.head_rows * D + c;
            const int last = min(lim, (it.tile + it.cnt) * kTcKeys - 1);
#pragma unroll 1
            for (int k = max(tc_seen_by_all(a, it.flat, len) + 1, it.tile * kTcKeys); k <= last; ++k) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(vr + static_cast<int64_t>(k) * D + e);
                add_not_finite(x.x, o[e], o[e + 1]);
                add_not_finite(x.y, o[e + 2], o[e + 3]);
                add_not_finite(x.z, o[e + 4], o[e + 5]);
                add_not_finite(x.w, o[e + 6], o[e + 7]);
              }
            }
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + sw128_off(lane, (c >> 3 & 4) + e)) =
                  make_uint4(pack_bf16x2(o[8 * e], o[8 * e + 1]), pack_bf16x2(o[8 * e + 2], o[8 * e + 3]),
                             pack_bf16x2(o[8 * e + 4], o[8 * e + 5]), pack_bf16x2(o[8 * e + 6], o[8 * e + 7]));
            if (!(c & 32)) continue;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(stage + sw128_off(lane, e)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = 4 * i + rsub;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + sw128_off(rr, csub));
            const int64_t out_row = __shfl_sync(0xffffffffu, row, rr);
            if (!(on_rows >> rr & 1)) continue;
            if (whole) *reinterpret_cast<uint4*>(a.out + out_row * D + (c & ~63) + 8 * csub) = v;
            else *reinterpret_cast<uint4*>(a.part_o + (pr + rr) * D + c + 4 * csub) = v;
          }
        }
        if (!ok) break;
        if (on && (pair || s == 0)) {
          if (!whole) a.part_ml[pr + lane] = make_float2(ref, l);
          else if (a.lse2) a.lse2[(static_cast<int64_t>(b) * a.nkv + it.kvh) * rows + r] = l == 0.f ? INFINITY : ref + log2f(l);
        }
        __syncwarp();
      }
      it = nx;
    }
    // items whose rows see nothing are in no worker's range
    if (ok && a.direct)
      for (int f = blockIdx.x; f < a.items(); f += gridDim.x) {
        if (a.tiles(f) > 0) continue;
        const int b = a.by_rps.divide(f), row_base = (f - b * a.rps) * kTcRows, n = min(rows - row_base, kTcRows);
        for (int i = threadIdx.x; i < n * a.nkv * (D / 8); i += kMmaWarp * 32) {
          const int ch = i % (D / 8), rk = i / (D / 8), kvh = rk / n, r = row_base + rk - kvh * n, tk = r / a.group;
          *reinterpret_cast<uint4*>(a.out + ((static_cast<int64_t>(b) * a.L + tk) * a.nh + kvh * a.group + r - tk * a.group) * D +
                                    8 * ch) = make_uint4(0, 0, 0, 0);
          if (ch == 0 && a.lse2) a.lse2[(static_cast<int64_t>(b) * a.nkv + kvh) * rows + r] = INFINITY;
        }
      }
  } else if (warp < kMmaWarp + 2) {
    // ---------------------------------------------------------------- MMA issuers
    // elect.sync, not a lane test: one lane chosen so lets the compiler hold the operands in uniform
    // registers (65 to 90 cycles a product otherwise, where the pipe takes 48)
    if (elect_one()) {
      const int s = warp - kMmaWarp;
      const uint64_t q_desc = sdesc_sw128(smem_u32(s_q)), k_desc = sdesc_sw128(smem_u32(s_kv));
      const uint64_t v_desc = sdesc_mn_sw128(smem_u32(s_kv), kTcKeys * 128);
      constexpr uint32_t kTile16 = S::kTileBytes >> 4;      // in descriptor units
      constexpr uint32_t kHalf16 = kTcKeys * 128 >> 4;      // the next 64 columns of a tile
      constexpr uint32_t kStep16 = kStep * 128 >> 4;        // the next 64 keys
      const uint32_t id_s = idesc_bf16(kTcKeys, kStep), id_o = idesc_bf16(kTcKeys, D) | (1u << 16);  // B MN-major
      const uint32_t t_s = tmem + s * kTcKeys, t_o = tmem + 2 * kTcKeys + s * D;
      int qph = 0, kslot = 0, vslot = 0, ring = 0;
      uint32_t ring_ph = 0, g = 0;  // g: steps done by the stream, as there
      bool ok = true;
      auto next_slot = [&](int& slot) {
        slot = ring;
        const bool got = mbar_wait(&bars.kvfull[slot], ring_ph, abort_flag, a.err);
        if (++ring == NS) {
          ring = 0;
          ring_ph ^= 1;
        }
        return got;
      };
      for (; ok && it.cnt > 0; tc_next(a, it)) {
        // with one row tile a tile is one step, the stream's half of its keys
        const bool pair = rows - (it.flat - a.by_rps.divide(it.flat) * a.rps) * kTcRows > kTcKeys;
        const int steps = pair ? 2 * it.cnt : it.cnt;
        const uint64_t ad = q_desc + (pair ? s : 0) * kTile16;
        auto issue_s = [&](int n) {
          const bool odd = pair && (n & 1);
          if (!odd && !next_slot(kslot)) return false;
          tc_fence_after();
          const uint64_t bd = k_desc + kslot * kTile16 + (pair ? n & 1 : s) * kStep16;
          const uint32_t buf = (g + n) & 1, d = t_s + buf * kStep;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(d, ad + (kk >> 2) * kHalf16 + 2 * (kk & 3), bd + (kk >> 2) * kHalf16 + 2 * (kk & 3), id_s, kk != 0);
          umma_commit(&bars.sfull[s][buf]);
          if (odd || !pair) umma_commit(&bars.kvempty[kslot]);
          return true;
        };
        for (int i = 0; ok && i < 2; ++i) ok = mbar_wait(&bars.qfull[i], qph & 1, abort_flag, a.err);
        ++qph;
        tc_fence_after();
        for (int n = 0; ok && n < min(2, steps); ++n) ok = issue_s(n);
#pragma unroll 1
        for (int n = 0; ok && n < steps; ++n) {
          const uint32_t buf = (g + n) & 1;
          const bool odd = pair && (n & 1);
          if (!odd) ok = next_slot(vslot);
          ok = ok && mbar_wait(&bars.pfull[s][buf], (g + n) >> 1 & 1, abort_flag, a.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t bd = v_desc + vslot * kTile16 + (pair ? n & 1 : s) * kStep16;
          const uint32_t at = t_s + buf * kStep;
#pragma unroll
          for (int kk = 0; kk < kStep / 16; ++kk) umma_bf16_ts(t_o, at + 8 * kk, bd + kk * 128, id_o, n != 0 || kk != 0);
          if (odd || !pair) umma_commit(&bars.kvempty[vslot]);
          if (n + 2 < steps) ok = issue_s(n + 2);
          else if (n + 2 == steps) umma_commit(&bars.otail[s]);
        }
        if (ok) umma_commit(&bars.ofull);
        g += steps;
      }
      // every product and commit of this lane has landed before the CTA frees TMEM and leaves
      umma_commit(&bars.done[s]);
      wait_drained(&bars.done[s], 0, a.err);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- K / V loader
    int kc = 0, tph = 0;
    bool ok = true;
    uint32_t piece = 0;
    for (; ok && it.cnt > 0; tc_next(a, it), ++piece) {
      const int b = a.by_rps.divide(it.flat);
      const bool pair = rows - (it.flat - b * a.rps) * kTcRows > kTcKeys;
      const int len = tc_len(a, b), sees = tc_seen_by_all(a, it.flat, len);
      const int y0 = (b * a.nkv + it.kvh) * a.head_rows;
      auto load = [&](const CUtensorMap* map, int j, bool v) {
        const int slot = kc % NS;
        if (!mbar_wait_lane0(&bars.kvempty[slot], ((kc / NS) & 1) ^ 1, abort_flag, a.err)) return false;
        ++kc;
        uint8_t* dst = s_kv + slot * S::kTileBytes;
        const int key0 = (it.tile + j) * kTcKeys;
        // Rows of V past the length may hold anything, and 0 * NaN is NaN: they become zeros.  So
        // do infinities and NaN in the rows that some of the item's tokens do not see (the streams
        // add them to the other tokens' output).
        const int first = max(sees + 1 - key0, 0), held = min(len - key0, kTcKeys);
        const bool ragged = v && (held < kTcKeys || first < held);
        uint64_t* bar = ragged ? &bars.tail : &bars.kvfull[slot];
        if (elect_one()) {
          mbar_arrive_expect_tx(bar, S::kTileBytes);
#pragma unroll
          for (int h = 0; h < S::kHalf; ++h)
            tma_load_2d(smem_u32(dst) + h * (kTcKeys * 128), map, h * 64, y0 + key0, bar);
        }
        __syncwarp();
        if (ragged) {
          if (!__all_sync(0xffffffffu, wait_drained(&bars.tail, tph & 1, a.err))) return false;
          ++tph;
          auto chunk = [&](int row, int e, int h) {
            return reinterpret_cast<uint4*>(dst + h * (kTcKeys * 128) + (row + (e >> 3)) * 128 + (e & 7) * 16);
          };
          bool bad = false;
          for (int e = lane; e < (held - first) * 8; e += 32)
#pragma unroll
            for (int h = 0; h < S::kHalf; ++h) {
              uint4* p = chunk(first, e, h);
              const uint4 x = *p;
              const uint4 y = make_uint4(finite_or_zero(x.x), finite_or_zero(x.y), finite_or_zero(x.z), finite_or_zero(x.w));
              if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                bad = true;
                *p = y;
              }
            }
          if (__any_sync(0xffffffffu, bad) && lane == 0)
            *const_cast<volatile uint32_t*>(&bars.hidden[piece & 7]) = piece + 1;
          for (int e = lane; e < (kTcKeys - held) * 8; e += 32)
#pragma unroll
            for (int h = 0; h < S::kHalf; ++h) *chunk(held, e, h) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.kvfull[slot]);
        }
        return true;
      };
      // in the order of their first use: K0 V0 K1 V1 .. (pair), K0 K1 V0 K2 V1 .. (one tile)
      if (!pair) {
        ok = load(&map_k, 0, false);
        if (ok && it.cnt > 1) ok = load(&map_k, 1, false);
      }
      for (int j = 0; ok && j < it.cnt; ++j) {
        if (pair) ok = load(&map_k, j, false);
        ok = ok && load(&map_v, j, true);
        if (ok && !pair && j + 2 < it.cnt) ok = load(&map_k, j + 2, false);
      }
    }
    // copies in flight land before the CTA leaves (all did unless a wait ran out)
    if (!ok)
      for (int j = max(0, kc - NS); j < kc; ++j)
        if (!wait_drained(&bars.kvfull[j % NS], (j / NS) & 1, a.err)) break;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ slot weights
// acc[j] of a kv head's 128 keys: S^T = K Q^T for 128 query rows at a time (keys are the TMEM
// lanes, rows the columns), so a thread's sum over its columns of 2^(s - lse of the row) is its
// key's weight and needs no other thread.  The four groups of 128 threads take every fourth row
// tile (two groups were bound by latency: 44% of the issue slots).  Bound by the
// exponentials (128 x 128 a tile: 1024 cycles of the special-function units against 512 of the
// tensor pipe).
//   warps 0-15  groups 0-3     warp 16  MMA issuer     warp 17  TMA loads of K and Q
namespace {
constexpr int kWThreads = 576;
constexpr int kWMmaWarp = 16;
constexpr int kWStages = kTcWeightParts;  // Q tiles, TMEM buffers, groups; twice as many rows' lse, which
                                          // the sums read after the product has freed its Q tile

template <int D>
struct WShape {
  static constexpr uint32_t kTileBytes = kTcKeys * D * 2;
  static constexpr uint32_t kSmem = 1024 + (2 + kWStages) * kTileBytes;
};

struct WBars {
  uint64_t qfull[kWStages], qempty[kWStages], sfull[kWStages], sempty[kWStages], kfull[2], kempty[2], done;
  uint32_t tmem;
  int abort_flag;
};
}  // namespace

template <int D>
__global__ void __launch_bounds__(kWThreads, 1) slot_weight_tc_kernel(const __grid_constant__ TcWeightArgs a,
                                                                     const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_q) {
  using S = WShape<D>;
  extern __shared__ uint8_t s_raw[];
  __shared__ WBars bars;
  __shared__ __align__(16) float s_lse[2 * kWStages][kTcKeys];  // negated; -inf: no such row
  const uint32_t pad = (1024u - (smem_u32(s_raw) & 1023u)) & 1023u;
  uint8_t* s_k = s_raw + pad;                    // [2][kTileBytes]
  uint8_t* s_q = s_k + 2 * S::kTileBytes;        // [kWStages][kTileBytes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars.abort_flag;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWStages; ++i) {
      mbar_init(&bars.qfull[i], 2);  // the copy, and the rows' lse
      mbar_init(&bars.qempty[i], 1);
      mbar_init(&bars.sfull[i], 2);  // the product, and its issuer (for the loader's writes of lse)
      mbar_init(&bars.sempty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.kfull[i], 1);
      mbar_init(&bars.kempty[i], 1);
    }
    mbar_init(&bars.done, 1);
    bars.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  // rows past a Q tile's whole tokens are never copied: zeros
  for (uint32_t i = threadIdx.x; i < kWStages * S::kTileBytes / 16; i += kWThreads)
    reinterpret_cast<uint4*>(s_q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  if (warp == kWMmaWarp) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  pdl_wait();
  pdl_trigger();
  const int per = tc_places_per_worker(a, tc_places_before(a, a.items()) * a.nkv);
  TcPiece it;
  tc_first(a, blockIdx.x, per, it);
  const int rows = a.L * a.group;
  uint32_t t = 0;  // tiles of this CTA: tile t is in stage t % 4

  if (warp < kWMmaWarp) {
    // ---------------------------------------------------------------- sums
    const int grp = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int kl = (warp & 3) * 32 + lane;
    bool ok = true;
    for (; ok && it.cnt > 0; tc_next(a, it)) {
      const int b = it.flat / a.key_tiles, key0 = (it.flat - b * a.key_tiles) * kTcKeys;
      const int len = a.lens[b];
      const int tile_rows = a.tile_tokens * a.group;
      const int row0 = (a.first_tile(key0, len) + it.tile) * tile_rows;
      // the first row that sees this lane's key; the item's last key's bounds the masked tiles
      const int tk = max(key0 + kl - (len - a.L), 0), tk_last = max(min(key0 + kTcKeys, len) - 1 - (len - a.L), 0);
      const int rmin = key0 + kl < len ? tk * a.group : 0x7fffffff, rmin_last = tk_last * a.group;
      float total = 0.f, low = 0.f;  // a compensated sum over tiles
      for (int i = 0; i < it.cnt; ++i, ++t) {
        const uint32_t st = t % kWStages;
        if (st != static_cast<uint32_t>(grp)) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.sfull[st], t / kWStages & 1, abort_flag, a.err))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int r0 = row0 + i * tile_rows;
        // a copy past the sequence's tokens brings another's rows
        const bool masked = r0 < rmin_last || r0 + tile_rows > rows;
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int c = 0; c < kTcKeys; c += 32) {
          float v[32];
          tmem_ld32_async(tmem + lanes + st * kTcKeys + c, v);
          tmem_wait_ld();
          if (c + 32 > tile_rows) {  // columns past the tile's rows: zeros, but NaN where a key is infinite
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c + e >= tile_rows) v[e] = 0.f;
          }
          const float4* nl = reinterpret_cast<const float4*>(&s_lse[t % (2 * kWStages)][c]);
          if (masked) {  // after lse, which may be NaN: such a row has no weight on what it does not see
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 n4 = nl[e];
              const float n[4] = {n4.x, n4.y, n4.z, n4.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = r0 + c + 4 * e + i;
                const float x = fmaf(v[4 * e + i], a.scale_log2, n[i]);
                sum4[i] += ex2(r >= rmin && r < rows ? x : -INFINITY);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 n4 = nl[e];
              sum4[0] += ex2(fmaf(v[4 * e], a.scale_log2, n4.x));
              sum4[1] += ex2(fmaf(v[4 * e + 1], a.scale_log2, n4.y));
              sum4[2] += ex2(fmaf(v[4 * e + 2], a.scale_log2, n4.z));
              sum4[3] += ex2(fmaf(v[4 * e + 3], a.scale_log2, n4.w));
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.sempty[st]);
        const float y = ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])) - low, u = total + y;
        low = (u - total) - y;
        total = u;
      }
      if (!ok) break;
      a.part[(tc_slot(a, blockIdx.x, it) * kTcWeightParts + grp) * kTcKeys + kl] = total;
    }
  } else if (warp == kWMmaWarp) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      const uint64_t k_desc = sdesc_sw128(smem_u32(s_k)), q_desc = sdesc_sw128(smem_u32(s_q));
      constexpr uint32_t kTile16 = S::kTileBytes >> 4, kHalf16 = kTcKeys * 128 >> 4;
      const uint32_t id = idesc_bf16(kTcKeys, kTcKeys);
      bool ok = true;
      uint32_t n = 0;  // items
      for (; ok && it.cnt > 0; tc_next(a, it), ++n) {
        ok = mbar_wait(&bars.kfull[n & 1], n >> 1 & 1, abort_flag, a.err);
#pragma unroll 1
        for (int i = 0; ok && i < it.cnt; ++i, ++t) {
          const uint32_t st = t % kWStages;
          ok = mbar_wait(&bars.qfull[st], t / kWStages & 1, abort_flag, a.err) &&
               mbar_wait(&bars.sempty[st], (t / kWStages & 1) ^ 1, abort_flag, a.err);
          if (!ok) break;
          mbar_arrive(&bars.sfull[st]);
          tc_fence_after();
          const uint64_t ad = k_desc + (n & 1) * kTile16, bd = q_desc + st * kTile16;
          const uint32_t d = tmem + st * kTcKeys;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(d, ad + (kk >> 2) * kHalf16 + 2 * (kk & 3), bd + (kk >> 2) * kHalf16 + 2 * (kk & 3), id, kk != 0);
          umma_commit(&bars.sfull[st]);
          umma_commit(&bars.qempty[st]);
        }
        if (ok) umma_commit(&bars.kempty[n & 1]);
      }
      umma_commit(&bars.done);
      wait_drained(&bars.done, 0, a.err);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- loader
    const int tile_rows = a.tile_tokens * a.group;
    const uint32_t tile_bytes = static_cast<uint32_t>(tile_rows) * 128;  // of a 64-column half
    bool ok = true;
    uint32_t n = 0;  // items
    for (; ok && it.cnt > 0; tc_next(a, it), ++n) {
      const int b = it.flat / a.key_tiles, key0 = (it.flat - b * a.key_tiles) * kTcKeys;
      const int tile0 = a.first_tile(key0, a.lens[b]) + it.tile;
      if (!mbar_wait_lane0(&bars.kempty[n & 1], (n >> 1 & 1) ^ 1, abort_flag, a.err)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&bars.kfull[n & 1], S::kTileBytes);
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
          tma_load_2d(smem_u32(s_k + (n & 1) * S::kTileBytes) + h * (kTcKeys * 128), &map_k, h * 64,
                      (b * a.nkv + it.kvh) * a.max_len + key0, &bars.kfull[n & 1]);
      }
      __syncwarp();
      const float* lse = a.lse2 + (static_cast<int64_t>(b) * a.nkv + it.kvh) * rows;
      float nl[4];
      auto fetch = [&](int i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 32 * e + lane, r = (tile0 + i) * tile_rows + c;
          nl[e] = c < tile_rows && r < rows ? -lse[r] : -INFINITY;
        }
      };
      fetch(0);
      for (int i = 0; i < it.cnt; ++i, ++t) {
        const uint32_t st = t % kWStages;
        // the product of tile t - 4 is complete; it waited for the sums of tile t - 8, so their
        // rows' lse are free too
        if (!mbar_wait_lane0(&bars.qempty[st], (t / kWStages & 1) ^ 1, abort_flag, a.err)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(&bars.qfull[st], tile_bytes * (D / 64));
#pragma unroll
          for (int h = 0; h < D / 64; ++h)
            tma_load_3d(smem_u32(s_q + st * S::kTileBytes) + h * (kTcKeys * 128), &map_q, h * 64, it.kvh * a.group,
                        b * a.L + (tile0 + i) * a.tile_tokens, &bars.qfull[st]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s_lse[t % (2 * kWStages)][32 * e + lane] = nl[e];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.qfull[st]);
        if (i + 1 < it.cnt) fetch(i + 1);
      }
    }
    // copies in flight land before the CTA leaves (their products waited for them unless a wait
    // ran out)
    if (*abort_flag) {
      for (uint32_t j = t > kWStages ? t - kWStages : 0; j < t; ++j) wait_drained(&bars.qfull[j % kWStages], j / kWStages & 1, a.err);
      if (n > 0) wait_drained(&bars.kfull[(n - 1) & 1], (n - 1) >> 1 & 1, a.err);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
static cudaError_t tc_opt_in() {
  const cudaError_t e = cudaFuncSetAttribute(attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(slot_weight_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, WShape<D>::kSmem);
}

cudaError_t attn_tc_init() {
  const cudaError_t e = tc_opt_in<128>();
  return e == cudaSuccess ? tc_opt_in<64>() : e;
}

cudaError_t launch_slot_weight_tc(const TcWeightArgs& a, int d, const CUtensorMap& k, const CUtensorMap& q, cudaStream_t st) {
  return d == 128 ? launch_pdl(slot_weight_tc_kernel<128>, a.workers, kWThreads, WShape<128>::kSmem, st, a, k, q)
                  : launch_pdl(slot_weight_tc_kernel<64>, a.workers, kWThreads, WShape<64>::kSmem, st, a, k, q);
}

cudaError_t launch_attn_tc(const TcAttnArgs& a, int d, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  return d == 128 ? launch_pdl(attn_tc_kernel<128>, a.workers, kThreads, Shape<128>::kSmem, st, a, k, v)
                  : launch_pdl(attn_tc_kernel<64>, a.workers, kThreads, Shape<64>::kSmem, st, a, k, v);
}

}  // namespace fm
