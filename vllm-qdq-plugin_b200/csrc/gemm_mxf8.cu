// MXFP8 products on the sm_100a tensor cores (tcgen05 kind::mxf8f6f4):
//   dense    C[m, n] = sum_k A[m, k] W[n, k] (+ bias[n])
//   grouped  C[s, n] = sum_k A[s / top_k, k] W_e[n, k] (x topk_weights[s])
//            for the slots s of the blocks of expert e
// A and W are E4M3 codes with one E8M0 scale per 32 elements of K; fp32
// accumulation, one rounding to the 16-bit output.
//
// The MMA's M side is 128 rows of W and its N side the activation rows
// ("swap AB"), so that few activation rows make a narrow N instead of an
// idle M, and a ragged segment of an expert's rows costs its own width.
//
// One CTA per SM walks work items (a segment of at most NT activation rows,
// 128 rows of W); 14 warps:
//   warp 0      TMA producer: W codes and scales of a K-128 stage, and the
//               codes of the segment's rows, which are consecutive (grouped:
//               a pass before copies the routed rows into sorted order)
//   warp 1      MMA issuer: per stage 4 MMAs (K = 32 each), M = 128,
//               N = the segment's rows rounded up to 16
//   warps 2-5   activation scales, four stages ("quad") at a time into a ring
//               of four quads, one per warp: a lane loads 16 scales of a row
//               at once and writes each stage's four bytes into the chunk
//               layout that tcgen05.cp expects.  One proxy fence a quad: a
//               fence per stage held the whole ring to 0.55 us a stage
//   warps 6-13  epilogue: TMEM lanes = W rows, columns = activation rows
// Scale bytes behind K / 32 (the rows' padding) are masked: their codes are
// zeros, but zero times a stale NaN scale would not be.
// What the kernel before it on the stream may have written (scales, routing,
// segments) is read past L1 (__ldcg): under programmatic dependent launch this
// kernel's CTAs start before that one has finished.
// The stage ring runs across items and the accumulator is double-buffered in
// TMEM, so an item's epilogue overlaps the next item's MMAs.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "mx_quant.cuh"
#include "sm100.cuh"

namespace qdqb200 {
namespace {

using namespace sm100;

constexpr int TM = 128;              // W rows per item (UMMA M)
constexpr int TK = 128;              // K elements (= bytes) per stage: one swizzle row
constexpr int NT_MAX = 192;          // activation rows per item: two accumulators + scales fit 512 TMEM columns
constexpr int T_W = TM * TK;         // 16 KB
constexpr int T_STAGES_MAX = 12;
constexpr int T_EPI = 8;             // epilogue warps
constexpr int T_SCALE = 4;           // scale warps = quads of stages in the scale ring
constexpr int T_THREADS = 32 * (2 + T_SCALE + T_EPI);
constexpr uint32_t T_TMEM = 512, T_SFW = 2 * NT_MAX, T_SFA = T_SFW + 4;
constexpr uint32_t T_SF_COLS = 12;   // a set of scale columns for each stage of a quad (one or two sets in turn: the same times)

__host__ __device__ constexpr int t_stage_bytes(int nt) { return T_W + nt * TK; }       // codes
__host__ __device__ constexpr int t_sf_bytes(int nt) { return nt > 128 ? 1024 : 512; }  // a stage's activation scales
__host__ __device__ constexpr int t_quads_bytes(int nt) { return 4 * T_SCALE * (t_sf_bytes(nt) + 512); }

struct __align__(8) TBars {
  uint64_t full[T_STAGES_MAX];   // codes and W scales landed (1 arrival + tx)
  uint64_t empty[T_STAGES_MAX];  // the stage's MMAs completed
  uint64_t sf_full[T_SCALE];     // a quad's activation scales are written, its W scales landed (2 arrivals + tx)
  uint64_t sf_empty[T_SCALE];    // the quad's MMAs completed
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
constexpr int kSmemMax = 227 * 1024;
constexpr int T_OUT = 16 * TM * 2;  // an epilogue half's output rows on their way out
__host__ __device__ constexpr int t_stages(int nt) {
  const int n = (kSmemMax - 1024 - static_cast<int>(sizeof(TBars)) - t_quads_bytes(nt) - 2 * T_OUT) / t_stage_bytes(nt);
  return n < T_STAGES_MAX ? n : T_STAGES_MAX;
}
__host__ __device__ constexpr int t_smem(int nt) {
  return 1024 + t_stages(nt) * t_stage_bytes(nt) + t_quads_bytes(nt) + 2 * T_OUT + static_cast<int>(sizeof(TBars));
}

template <int kDtype>
struct Out16 {
  using T = __nv_bfloat16;
  __device__ static float load(const T* p) { return __bfloat162float(*p); }
  __device__ static T one(float a) { return __float2bfloat16_rn(a); }
  __device__ static uint32_t two(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Out16<QDQ_DTYPE_FP16> {
  using T = __half;
  __device__ static float load(const T* p) { return __half2float(*p); }
  __device__ static T one(float a) { return __float2half_rn(a); }
  __device__ static uint32_t two(float a, float b) { return pack_f16x2(a, b); }
};

// E4M3 codes of a 16-byte chunk of a 32-group with scale exponent e.
template <int kDtype>
__device__ __forceinline__ uint2 chunk_codes(const uint4& v, int e, float zero) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[2];
  mx8_codes<kDtype>(w, e, zero, c);
  return make_uint2(c[0], c[1]);
}

struct GemmArgs {
  const uint8_t* sfw;          // tiled W scales
  int64_t sf_per_expert;
  const uint8_t* sfa;          // row-major activation scales
  int64_t lds;
  const void* bias;            // dense
  void* c;
  int64_t ldc;
  const int32_t* seg_tab;      // grouped: [count, -, -, -], then (first position, rows, expert, -) per segment
  const int32_t* sorted_ids;
  const float* topk_w;         // nullptr: no scaling
  int M, N, K, kchunks;        // M: dense rows, grouped slots (size_m * top_k)
  int num_blocks, num_experts;
  int a_rows;                  // rows of the activation codes (grouped: sorted positions)
  int nt, box;                 // activation rows per item, and per TMA box
  int wide;                    // neighbouring n that C takes in one store: 8, 2 or 1
  int* status;
};

// Position in a ring of n slots and the phase parity of the current lap.  The
// depths are run-time values: dividing a running count by them cost the single
// issuing thread half of a stage's time.
struct Cursor {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// The scale bytes of K-128 stage kt that lie inside K.
__device__ __forceinline__ uint32_t scale_mask(int K, int kt) {
  const int valid = max(K / 32 - 4 * kt, 0);
  return valid >= 4 ? 0xFFFFFFFFu : (1u << (8 * valid)) - 1u;
}

template <int kR>
__device__ __forceinline__ void mask_quad(uint4 (&v)[kR], int K, int kt) {
#pragma unroll
  for (int j = 0; j < kR; ++j) {
    v[j].x &= scale_mask(K, kt);
    v[j].y &= scale_mask(K, kt + 1);
    v[j].z &= scale_mask(K, kt + 2);
    v[j].w &= scale_mask(K, kt + 3);
  }
}

struct Item {
  int row0;     // first activation row (dense) or first sorted position (grouped)
  int rows;     // rows of the segment; 0: nothing to do
  int n_tile;
  int expert;
};

// Walks a CTA's work items; every role decodes them alike.  Dense: tiles of
// one W panel run side by side, so the CTAs in flight share it in L2.
// Grouped: segment-major, so that each expert's W streams from HBM once while
// its rows stay in L2; the next item's segment entry is fetched while the
// present item runs.
template <bool kGrouped>
struct Walk {
  const GemmArgs& p;
  const int n_tiles, num_m, items, step;
  int i;
  int4 next;

  __device__ __forceinline__ Walk(const GemmArgs& args, int first, int stride, int tiles)
      : p(args), n_tiles(tiles), num_m(kGrouped ? 1 : (args.M + args.nt - 1) / args.nt),
        items(kGrouped ? min(max(__ldcg(args.seg_tab), 0), args.num_blocks) * tiles : num_m * tiles), step(stride),
        i(first - stride) {
    fetch(first);
  }
  __device__ __forceinline__ void fetch(int j) {
    if (kGrouped && j < items) next = __ldcg(reinterpret_cast<const int4*>(p.seg_tab + 4) + j / n_tiles);
  }
  __device__ __forceinline__ bool advance(Item& it) {
    i += step;
    if (i >= items) return false;
    if (kGrouped) {
      it = {next.x, next.y, i % n_tiles, next.z};
      // a malformed entry is nothing to do
      if (it.row0 < 0 || it.rows < 0 || it.rows > p.nt || it.row0 + it.rows > p.a_rows || it.expert < 0 ||
          it.expert >= p.num_experts)
        it.rows = 0;
      fetch(i + step);
    } else {
      it.n_tile = i / num_m;
      it.row0 = (i - it.n_tile * num_m) * p.nt;
      it.rows = min(p.nt, p.M - it.row0);
      it.expert = 0;
    }
    return true;
  }
};

// Output row of each of an item's columns (-1: none) and its factor, held by
// lane l for column 32 c + l.
template <bool kGrouped>
__device__ __forceinline__ void column_rows(const GemmArgs& p, const Item& w, int c, int lane, int& slot, float& wt) {
  const int col = 32 * c + lane;
  slot = -1;
  wt = 1.0f;
  if (col < w.rows) slot = kGrouped ? __ldcg(p.sorted_ids + w.row0 + col) : w.row0 + col;
  if (slot >= p.M) slot = -1;
  if (kGrouped && p.topk_w != nullptr && slot >= 0) wt = __ldcg(p.topk_w + slot);
}

// Where the output goes: copies in registers (behind a barrier's memory clobber
// every field of the kernel's arguments would be loaded again).
struct Target {
  void* c;
  int64_t ldc;
  int n, wide;
  bool biased, scaled;
  __device__ explicit Target(const GemmArgs& p)
      : c(p.c), ldc(p.ldc), n(p.N), wide(p.wide), biased(p.bias != nullptr), scaled(p.topk_w != nullptr) {}
};

// The output rows of 16 columns from shared memory, whole rows of 128 n at a
// time by the half's four warps: kWidth neighbouring n a store, up to four
// stores' words read before the first of them.
template <int kWidth, typename T>
__device__ __forceinline__ void store_rows(const Target& to, const uint8_t* out, int n0, int t, int slot, int first) {
  using Word = std::conditional_t<kWidth == 8, uint4, std::conditional_t<kWidth == 2, uint32_t, uint16_t>>;
  constexpr int kUnits = TM / kWidth, kRows = 128 / kUnits;  // stores a row, rows a pass
  constexpr int kPasses = 16 / kRows, kBatch = kPasses < 4 ? kPasses : 4;
  const int j = t % kUnits * kWidth, n = n0 + j;  // N is a multiple of kWidth
#pragma unroll
  for (int i0 = 0; i0 < kPasses; i0 += kBatch) {
    Word x[kBatch];
    int row[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = (i0 + i) * kRows + t / kUnits;
      row[i] = __shfl_sync(0xffffffffu, slot, first + r);
      x[i] = *reinterpret_cast<const Word*>(out + r * (2 * TM) + (((j >> 3) ^ (r & 7)) << 4) + (j & 7) * 2);
    }
    if (n < to.n) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (row[i] >= 0)
          *reinterpret_cast<Word*>(static_cast<T*>(to.c) + static_cast<int64_t>(row[i]) * to.ldc + n) = x[i];
    }
  }
}

// Stores 32 accumulator columns (activation rows) of the tile's 128 W rows n0..:
// the four warps of an epilogue half hold 32 W rows each as 8x8 fragments, which
// stmatrix transposes into rows of the output in shared memory (16 rows at a
// time; chunk j of row r lies at j ^ (r % 8), free of bank conflicts), and store
// whole lines from there: [4080 x 128] -> 9472 in 25.0 us, where filling the output
// takes 20.3.  (Transposed by shuffles in registers, 64 bytes of a row a store,
// 41; with the accumulator handed back by an arrival with release, which waits
// for the stores before it, 35.)
template <int kDtype, bool kGrouped>
__device__ __forceinline__ void store_columns(const Target& target, uint32_t (&acc)[32], uint8_t* out, int half, int q,
                                              int lane, int n0, int cols, int slot, float wt, const float (&bias)[4],
                                              bool store) {
  using O = Out16<kDtype>;
  const uint32_t to = smem_u32(out) + (lane & 7) * (2 * TM) + (((4 * q + (lane >> 3)) ^ (lane & 7)) << 4);
  // acc[16 h + 4 c + 2 g + e]: W row 16 h + 8 g + lane / 4 of the warp's, column 8 c + 2 (lane % 4) + e
  if (!kGrouped && target.biased) {
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = __float_as_uint(__uint_as_float(acc[i]) + bias[(i >> 4) * 2 + ((i >> 1) & 1)]);
  }
  if (kGrouped && target.scaled) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = __shfl_sync(0xffffffffu, wt, 8 * c + 2 * (lane & 3) + e);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t& x = acc[(g >> 1) * 16 + 4 * c + 2 * (g & 1) + e];
          x = __float_as_uint(__uint_as_float(x) * f);
        }
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (16 * s >= cols) break;
    uint32_t v[2][4];  // columns 16 s + 8 i .. + 7, W rows 8 g .. + 7 of the warp's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t* a = acc + (g >> 1) * 16 + 4 * (2 * s + i) + 2 * (g & 1);
        v[i][g] = O::two(__uint_as_float(a[0]), __uint_as_float(a[1]));
      }
    }
    named_barrier(1 + half, 128);  // the rows before have been read
#pragma unroll
    for (int i = 0; i < 2; ++i) stmatrix_x4_trans(to + i * 8 * (2 * TM), v[i]);
    named_barrier(1 + half, 128);
    if (store) {
      const int t = 32 * q + lane;
      if (target.wide == 8) store_rows<8, typename O::T>(target, out, n0, t, slot, 16 * s);
      else if (target.wide == 2) store_rows<2, typename O::T>(target, out, n0, t, slot, 16 * s);
      else store_rows<1, typename O::T>(target, out, n0, t, slot, 16 * s);
    }
  }
}

// The bias of a lane's four W rows n + 8 g + lane / 4 of the warp's 32.
template <int kDtype>
__device__ __forceinline__ void fragment_bias(const GemmArgs& p, int n, int lane, float (&bias)[4]) {
  using O = Out16<kDtype>;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = n + 8 * g + (lane >> 2);
    bias[g] = p.bias != nullptr && at < p.N ? O::load(static_cast<const typename O::T*>(p.bias) + at) : 0.f;
  }
}

template <int kDtype, bool kGrouped>
__global__ void __launch_bounds__(T_THREADS, 1)
mxf8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                 const __grid_constant__ GemmArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // code stages | quads of W scales | quads of activation scales | output rows | barriers
  const int S = t_stages(p.nt), stage_bytes = T_W + p.nt * TK, sf_bytes = t_sf_bytes(p.nt);
  uint8_t* s_sfw = smem + S * stage_bytes;
  uint8_t* s_sfa = s_sfw + 4 * T_SCALE * 512;
  uint8_t* s_out = s_sfa + 4 * T_SCALE * sf_bytes;
  TBars* bars = reinterpret_cast<TBars*>(s_out + 2 * T_OUT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n_tiles = (p.N + TM - 1) / TM;
  const int num_kt = (p.K + TK - 1) / TK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < T_SCALE; ++b) {
      mbar_init(&bars->sf_full[b], 2);
      mbar_init(&bars->sf_empty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 32 * T_EPI);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_a);
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, T_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);  // uniform
  Walk<kGrouped> walk(p, blockIdx.x, gridDim.x, n_tiles);
  Item w;

  if (warp == 0) {
    // ---------------- producer.  The whole warp walks the loop, so that its addresses stay in uniform registers;
    // one lane issues.
    const bool leader = elect_one();
    Cursor at, sf_at;
    int issued = 0, quads = 0;
    bool ok = true;
    while (ok && walk.advance(w)) {
      if (w.rows == 0) continue;
      const int w_row = w.expert * p.N + w.n_tile * TM;
      const uint8_t* sfw = p.sfw + w.expert * p.sf_per_expert + static_cast<int64_t>(w.n_tile) * p.kchunks * 512;
      const int boxes = (w.rows + p.box - 1) / p.box;
      const uint32_t tx = T_W + boxes * p.box * TK;
      for (int kt = 0; kt < num_kt; ++kt, ++issued, at.next(S)) {
        const int s = at.slot;
        if ((kt & 3) == 0) {  // W scales, four stages at once
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->sf_empty[sf_at.slot], sf_at.phase ^ 1u, p.status, 0x609));
          if (!ok) break;
          if (leader) {
            const uint32_t bytes = 512u * min(4, num_kt - kt);
            mbar_arrive_expect_tx(&bars->sf_full[sf_at.slot], bytes);
            bulk_load(s_sfw + sf_at.slot * 2048, sfw + static_cast<int64_t>(kt) * 512, bytes, &bars->sf_full[sf_at.slot]);
          }
          sf_at.next(T_SCALE);
          ++quads;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[s], at.phase ^ 1u, p.status, 0x601));
        if (!ok) break;
        uint8_t* st = smem + s * stage_bytes;
        if (leader) {
          mbar_arrive_expect_tx(&bars->full[s], tx);
          tma_load_2d(st, &tmap_w, kt * TK, w_row, &bars->full[s]);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(st + T_W + b * p.box * TK, &tmap_a, kt * TK, w.row0 + b * p.box, &bars->full[s]);
        }
      }
    }
    if (!ok) bars->abort = 1;
    // every issued copy has landed before the CTA may exit
    for (int j = max(0, issued - S); j < issued; ++j) mbar_wait(&bars->full[j % S], (j / S) & 1, p.status, 0x602);
    for (int j = max(0, quads - T_SCALE); j < quads; ++j)
      mbar_wait(&bars->sf_full[j % T_SCALE], (j / T_SCALE) & 1, p.status, 0x60a);
  } else if (warp == 1) {
    // ---------------- MMA issuer (the whole warp walks, one lane issues).  Stages that are both full go out as a
    // pair: at few rows the loop around a stage costs more than its MMAs.
    const bool leader = elect_one();
    Cursor at, sf_at, acc_at;
    const uint64_t dw0 = smem_desc_sw128(smem), dsw0 = smem_desc_sf(s_sfw), dsa0 = smem_desc_sf(s_sfa);
    bool ok = true;
    while (ok && walk.advance(w)) {
      if (w.rows == 0) continue;
      const int n_mma = (w.rows + 15) / 16 * 16;
      const uint32_t idesc = idesc_mxf8(TM, n_mma);
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_empty[acc_at.slot], acc_at.phase ^ 1u, p.status, 0x603));
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + NT_MAX * acc_at.slot;
      auto stage = [&](int kt, int s) {
        const uint64_t dsa = dsa0 + ((sf_at.slot * 4 + (kt & 3)) * sf_bytes >> 4);
        const uint32_t sf = tmem + T_SF_COLS * (kt & 3);
        tmem_cp_sf(sf + T_SFW, dsw0 + ((sf_at.slot * 4 + (kt & 3)) * 512 >> 4));
        tmem_cp_sf(sf + T_SFA, dsa);
        if (n_mma > 128) tmem_cp_sf(sf + T_SFA + 4, dsa + (512 >> 4));
        const uint64_t dw = dw0 + (s * stage_bytes >> 4), da = dw + (T_W >> 4);
#pragma unroll
        for (uint32_t kk = 0; kk < 4; ++kk)  // K step kk reads scale byte kk of each row's four
          mma_mxf8(acc, dw + 2 * kk, da + 2 * kk, idesc_with_sf_ids(idesc, kk, kk), (sf + T_SFW) | (kk << 30),
                   (sf + T_SFA) | (kk << 30), (kt | kk) != 0);
        tc_commit(&bars->empty[s]);
      };
      for (int kt = 0; kt < num_kt;) {
        if ((kt & 3) == 0) ok = mbar_wait(&bars->sf_full[sf_at.slot], sf_at.phase, p.status, 0x608);
        const Cursor one = at;
        at.next(S);
        const Cursor two = at;
        const bool pair = ok && (kt & 1) == 0 && kt + 1 < num_kt &&
                          __all_sync(0xffffffffu, mbar_test2(&bars->full[one.slot], one.phase, &bars->full[two.slot], two.phase));
        if (!pair) ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->full[one.slot], one.phase, p.status, 0x604));
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          stage(kt, one.slot);
          if (pair) stage(kt + 1, two.slot);
        }
        if (pair) at.next(S);
        kt += pair ? 2 : 1;
        if ((kt & 3) == 0 || kt == num_kt) {
          if (leader) tc_commit(&bars->sf_empty[sf_at.slot]);
          sf_at.next(T_SCALE);
        }
      }
      if (!ok) break;
      if (leader) tc_commit(&bars->acc_full[acc_at.slot]);
      acc_at.next(2);
    }
    if (!ok) bars->abort = 1;
    if (leader) {
      tc_commit(&bars->drain);
      mbar_wait(&bars->drain, 0, p.status, 0x605);
    }
  } else if (warp < 2 + T_SCALE) {
    // ---------------- activation scales: warp u fills the quads u, u + 4, ... of the CTA's stages
    constexpr int kR = NT_MAX / 32;  // rows per lane
    const int u = warp - 2;
    const int quads = (num_kt + 3) / 4;
    int quad = 0;  // first quad of the item, counted over the CTA's items
    bool ok = true;
    while (ok && walk.advance(w)) {
      if (w.rows == 0) continue;
      const int n_mma = (w.rows + 15) / 16 * 16;
      const uint8_t* src[kR];
#pragma unroll
      for (int j = 0; j < kR; ++j)
        src[j] = p.sfa + static_cast<int64_t>(min(w.row0 + lane + 32 * j, p.a_rows - 1)) * p.lds;
      for (int h = (u - quad) & (T_SCALE - 1); h < quads; h += T_SCALE) {
        uint4 v[kR];
#pragma unroll
        for (int j = 0; j < kR; ++j)
          if (lane + 32 * j < n_mma) v[j] = __ldcg(reinterpret_cast<const uint4*>(src[j] + 16 * h));
        if (h + 1 == quads) mask_quad(v, p.K, 4 * h);
        ok = mbar_wait(&bars->sf_empty[u], (((quad + h) / T_SCALE) & 1) ^ 1, p.status, 0x606);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* sf = s_sfa + u * 4 * sf_bytes;
#pragma unroll
        for (int j = 0; j < kR; ++j) {
          const int r = lane + 32 * j;
          if (r < n_mma) {
            uint8_t* at = sf + (j >> 2) * 512 + lane * 16 + (j & 3) * 4;
            *reinterpret_cast<uint32_t*>(at) = v[j].x;
            *reinterpret_cast<uint32_t*>(at + sf_bytes) = v[j].y;
            *reinterpret_cast<uint32_t*>(at + 2 * sf_bytes) = v[j].z;
            *reinterpret_cast<uint32_t*>(at + 3 * sf_bytes) = v[j].w;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->sf_full[u]);
      }
      quad += quads;
    }
    if (!ok) bars->abort = 1;
  } else {
    // ---------------- epilogue: warp reads TMEM lanes 32 (warp % 4).., column chunks half, half + 2, ...
    const int q = warp & 3, half = (warp - 2 - T_SCALE) >> 2;
    uint8_t* out = s_out + half * T_OUT;
    const Target target(p);
    bool ok = true;
    int j = 0;
    while (walk.advance(w)) {
      if (w.rows == 0) continue;
      const int nchunks = (w.rows + 31) / 32;
      // output rows of this warp's columns, fetched while the MMAs run
      int slot;
      float wt;
      column_rows<kGrouped>(p, w, half, lane, slot, wt);
      const int n0 = w.n_tile * TM;
      float bias[4];
      fragment_bias<kDtype>(p, n0 + q * 32, lane, bias);
      const int buf = j & 1;
      if (ok) ok = mbar_wait(&bars->acc_full[buf], (j >> 1) & 1, p.status, 0x607);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + NT_MAX * buf;
      const bool store = __all_sync(0xffffffffu, ok && !*(volatile int*)&bars->abort);
      if (half >= nchunks) {
        tc_fence_before();
        mbar_arrive(&bars->acc_empty[buf]);
      }
#pragma unroll 1
      for (int c = half; c < nchunks; c += 2) {
        uint32_t r[32];
        tmem_ld_frag(taddr + 32 * c, r);
        tmem_ld_frag(taddr + (16u << 16) + 32 * c, r + 16);
        tmem_ld_wait();
        if (c + 2 >= nchunks) {  // this warp's last chunk of the item
          tc_fence_before();
          mbar_arrive(&bars->acc_empty[buf]);
        }
        const int rows = slot;
        const float factor = wt;
        column_rows<kGrouped>(p, w, c + 2, lane, slot, wt);  // the next chunk's
        store_columns<kDtype, kGrouped>(target, r, out, half, q, lane, n0, w.rows - 32 * c, rows, factor, bias, store);
      }
      ++j;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, T_TMEM);
  }
}

// ---------------------------------------------------------------------------
// Many rows: the same walk by pairs of CTAs (tcgen05 cta_group::2).
//
// What bounds the kernel above at many rows is operand delivery: an SM takes
// in about 80 bytes a cycle, and a 128 x 192 item needs 106 to keep its MMAs
// going.  A pair shares one 256 x NT item: each CTA holds 128 rows of W and
// half of the activation rows, and its MMAs read the other half from its
// peer's shared memory, so an SM takes in 66 bytes a cycle at NT = 240.
// Two accumulators of 240 columns and two sets of scale columns fill TMEM.
//
// Roles as above, in both CTAs, with these differences: TMA completes on the
// leader's (rank 0) barriers, the leader alone issues MMAs and its commits
// arrive in both CTAs; each CTA writes the scales of all the item's rows to
// its own shared memory, which its half of the MMA reads.
// ---------------------------------------------------------------------------
constexpr int P_NT_MAX = 240;
constexpr int P_STAGES_MAX = 11;
constexpr uint32_t P_SFW = 2 * P_NT_MAX, P_SFA = P_SFW + 4, P_SF_COLS = 12, P_SF_SETS = 2;
static_assert(P_SFW + P_SF_SETS * P_SF_COLS <= 512, "pair TMEM columns");

struct __align__(8) PBars {
  uint64_t full[P_STAGES_MAX];   // leader: both CTAs' codes landed (1 arrival + tx)
  uint64_t empty[P_STAGES_MAX];  // each CTA: the pair's MMAs on the stage completed
  uint64_t sf_full[T_SCALE];     // leader: both CTAs' scales of the quad are in place (3 arrivals + tx)
  uint64_t sf_empty[T_SCALE];    // each CTA
  uint64_t acc_full[2];          // each CTA
  uint64_t acc_empty[2];         // leader: both CTAs' epilogue warps have read the accumulator
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
__host__ __device__ constexpr int p_stage_bytes(int tok) { return T_W + tok * TK; }  // tok: token rows held by a CTA
constexpr int P_QUADS = 4 * T_SCALE * (1024 + 512);
__host__ __device__ constexpr int p_stages(int tok) {
  const int n = (kSmemMax - 1024 - static_cast<int>(sizeof(PBars)) - P_QUADS - 2 * T_OUT) / p_stage_bytes(tok);
  return n < P_STAGES_MAX ? n : P_STAGES_MAX;
}
__host__ __device__ constexpr int p_smem(int tok) {
  return 1024 + p_stages(tok) * p_stage_bytes(tok) + P_QUADS + 2 * T_OUT + static_cast<int>(sizeof(PBars));
}

template <int kDtype, bool kGrouped>
__global__ void __launch_bounds__(T_THREADS, 1)
mxf8_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                 const __grid_constant__ CUtensorMap tmap_sfw, const __grid_constant__ GemmArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // code stages | quads of W scales | quads of activation scales | output rows | barriers
  const int tok_rows = (p.nt / 2 + p.box - 1) / p.box * p.box;
  const int S = p_stages(tok_rows), stage_bytes = p_stage_bytes(tok_rows);
  uint8_t* s_sfw = smem + S * stage_bytes;
  uint8_t* s_sfa = s_sfw + 4 * T_SCALE * 512;
  uint8_t* s_out = s_sfa + 4 * T_SCALE * 1024;
  PBars* bars = reinterpret_cast<PBars*>(s_out + 2 * T_OUT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int n_tiles = (p.N + 2 * TM - 1) / (2 * TM);
  const int num_kt = (p.K + TK - 1) / TK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < T_SCALE; ++b) {
      mbar_init(&bars->sf_full[b], 3);
      mbar_init(&bars->sf_empty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * T_EPI);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_sfw);
  }
  if (warp == 0) {
    tmem_alloc_pair(&bars->tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // both CTAs' barriers are initialised and the TMEM is allocated
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);
  Walk<kGrouped> walk(p, blockIdx.x >> 1, gridDim.x >> 1, n_tiles);
  Item w;

  if (warp == 0) {
    // ---------------- producer (both CTAs): own W rows and own half of the activation rows
    const bool leader = elect_one();
    Cursor at, sf_at;
    int issued = 0, quads = 0;
    bool ok = true;
    while (ok && walk.advance(w)) {
      if (w.rows == 0) continue;
      const int half = (w.rows + 15) / 16 * 8;  // half of the MMA's N
      const int w_row = w.expert * p.N + w.n_tile * 2 * TM + static_cast<int>(rank) * TM;
      const int a_row = w.row0 + static_cast<int>(rank) * half;
      const int sf_row = w.expert * static_cast<int>(p.sf_per_expert / 512) + (2 * w.n_tile + static_cast<int>(rank)) * p.kchunks;
      const int boxes = (half + p.box - 1) / p.box;
      for (int kt = 0; kt < num_kt; ++kt, ++issued, at.next(S)) {
        const int s = at.slot;
        if ((kt & 3) == 0) {  // W scales, four stages at once
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->sf_empty[sf_at.slot], sf_at.phase ^ 1u, p.status, 0x801));
          if (!ok) break;
          if (leader) {
            if (rank == 0) mbar_arrive_expect_tx(&bars->sf_full[sf_at.slot], 2 * 2048);
            tma_load_2d_pair(s_sfw + sf_at.slot * 2048, &tmap_sfw, 0, sf_row + kt, cluster_addr(&bars->sf_full[sf_at.slot], 0));
          }
          sf_at.next(T_SCALE);
          ++quads;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[s], at.phase ^ 1u, p.status, 0x802));
        if (!ok) break;
        uint8_t* st = smem + s * stage_bytes;
        if (leader) {
          const uint32_t full0 = cluster_addr(&bars->full[s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * (T_W + boxes * p.box * TK));
          tma_load_2d_pair(st, &tmap_w, kt * TK, w_row, full0);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d_pair(st + T_W + b * p.box * TK, &tmap_a, kt * TK, a_row + b * p.box, full0);
        }
      }
    }
    if (!ok) bars->abort = 1;
    // The leader's barriers cover the pair's copies still in flight.
    if (rank == 0) {
      for (int j = max(0, issued - S); j < issued; ++j) mbar_wait(&bars->full[j % S], (j / S) & 1, p.status, 0x803);
      for (int j = max(0, quads - T_SCALE); j < quads; ++j)
        mbar_wait(&bars->sf_full[j % T_SCALE], (j / T_SCALE) & 1, p.status, 0x804);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader)
    if (rank == 0) {
      const bool leader = elect_one();
      Cursor at, sf_at, acc_at;
      const uint64_t dw0 = smem_desc_sw128(smem), dsw0 = smem_desc_sf(s_sfw), dsa0 = smem_desc_sf(s_sfa);
      bool ok = true;
      while (ok && walk.advance(w)) {
        if (w.rows == 0) continue;
        const int n_mma = (w.rows + 15) / 16 * 16;
        const uint32_t idesc = idesc_mxf8(2 * TM, n_mma);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_empty[acc_at.slot], acc_at.phase ^ 1u, p.status, 0x805));
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem + P_NT_MAX * acc_at.slot;
        for (int kt = 0; kt < num_kt; ++kt, at.next(S)) {
          const int s = at.slot;
          if ((kt & 3) == 0) ok = mbar_wait_cluster(&bars->sf_full[sf_at.slot], sf_at.phase, p.status, 0x806);
          ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->full[s], at.phase, p.status, 0x807));
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t dsa = dsa0 + ((sf_at.slot * 4 + (kt & 3)) * 1024 >> 4);
            const uint32_t sf = tmem + P_SF_COLS * (kt & (P_SF_SETS - 1));
            tmem_cp_sf_pair(sf + P_SFW, dsw0 + ((sf_at.slot * 4 + (kt & 3)) * 512 >> 4));
            tmem_cp_sf_pair(sf + P_SFA, dsa);
            if (n_mma > 128) tmem_cp_sf_pair(sf + P_SFA + 4, dsa + (512 >> 4));
            const uint64_t dw = dw0 + (s * stage_bytes >> 4), da = dw + (T_W >> 4);
#pragma unroll
            for (uint32_t kk = 0; kk < 4; ++kk)
              mma_mxf8_pair(acc, dw + 2 * kk, da + 2 * kk, idesc_with_sf_ids(idesc, kk, kk), (sf + P_SFW) | (kk << 30),
                            (sf + P_SFA) | (kk << 30), (kt | kk) != 0);
            tc_commit_pair(&bars->empty[s]);
            if ((kt & 3) == 3 || kt + 1 == num_kt) tc_commit_pair(&bars->sf_empty[sf_at.slot]);
          }
          if ((kt & 3) == 3 || kt + 1 == num_kt) sf_at.next(T_SCALE);
        }
        if (!ok) break;
        if (leader) tc_commit_pair(&bars->acc_full[acc_at.slot]);
        acc_at.next(2);
      }
      if (!ok) bars->abort = 1;
      if (leader) {
        tc_commit_pair_local(&bars->drain);  // tracks the pair's tcgen05 ops
        mbar_wait(&bars->drain, 0, p.status, 0x808);
      }
    }
  } else if (warp < 2 + T_SCALE) {
    // ---------------- activation scales of all the item's rows, in both CTAs
    constexpr int kR = (P_NT_MAX + 31) / 32;  // rows per lane
    const int u = warp - 2;
    const int quads = (num_kt + 3) / 4;
    const uint32_t full0 = cluster_addr(&bars->sf_full[u], 0);
    int quad = 0;
    bool ok = true;
    while (ok && walk.advance(w)) {
      if (w.rows == 0) continue;
      const int n_mma = (w.rows + 15) / 16 * 16;
      const uint8_t* src[kR];
#pragma unroll
      for (int j = 0; j < kR; ++j)
        src[j] = p.sfa + static_cast<int64_t>(min(w.row0 + lane + 32 * j, p.a_rows - 1)) * p.lds;
      for (int h = (u - quad) & (T_SCALE - 1); h < quads; h += T_SCALE) {
        uint4 v[kR];
#pragma unroll
        for (int j = 0; j < kR; ++j)
          if (lane + 32 * j < n_mma) v[j] = __ldcg(reinterpret_cast<const uint4*>(src[j] + 16 * h));
        if (h + 1 == quads) mask_quad(v, p.K, 4 * h);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->sf_empty[u], (((quad + h) / T_SCALE) & 1) ^ 1, p.status, 0x809));
        if (!ok) break;
        uint8_t* sf = s_sfa + u * 4 * 1024;
#pragma unroll
        for (int j = 0; j < kR; ++j) {
          if (lane + 32 * j < n_mma) {
            uint8_t* at = sf + (j >> 2) * 512 + lane * 16 + (j & 3) * 4;
            const uint32_t four[4] = {v[j].x, v[j].y, v[j].z, v[j].w};  // one word for each stage of the quad
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(at + i * 1024) = four[i];
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(full0);
      }
      quad += quads;
    }
    if (!ok) bars->abort = 1;
  } else {
    // ---------------- epilogue (both CTAs): TMEM lanes = the CTA's 128 W rows, columns = activation rows
    const int q = warp & 3, half = (warp - 2 - T_SCALE) >> 2;
    uint8_t* out = s_out + half * T_OUT;
    const Target target(p);
    Cursor acc_at;
    bool ok = true;
    while (walk.advance(w)) {
      if (w.rows == 0) continue;
      const int nchunks = (w.rows + 31) / 32;
      int slot;
      float wt;
      column_rows<kGrouped>(p, w, half, lane, slot, wt);
      const int n0 = (2 * w.n_tile + static_cast<int>(rank)) * TM;
      float bias[4];
      fragment_bias<kDtype>(p, n0 + q * 32, lane, bias);
      const uint32_t acc_empty0 = cluster_addr(&bars->acc_empty[acc_at.slot], 0);
      if (ok) ok = mbar_wait(&bars->acc_full[acc_at.slot], acc_at.phase, p.status, 0x80a);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + P_NT_MAX * acc_at.slot;
      const bool store = __all_sync(0xffffffffu, ok && !*(volatile int*)&bars->abort);
      if (half >= nchunks) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0);
      }
#pragma unroll 1
      for (int c = half; c < nchunks; c += 2) {
        uint32_t r[32];
        tmem_ld_frag(taddr + 32 * c, r);
        tmem_ld_frag(taddr + (16u << 16) + 32 * c, r + 16);
        tmem_ld_wait();
        if (c + 2 >= nchunks) {  // this warp's last chunk of the item
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0);
        }
        const int rows = slot;
        const float factor = wt;
        column_rows<kGrouped>(p, w, c + 2, lane, slot, wt);  // the next chunk's
        store_columns<kDtype, kGrouped>(target, r, out, half, q, lane, n0, w.rows - 32 * c, rows, factor, bias, store);
      }
      acc_at.next(2);
    }
  }

  // Neither CTA releases the pair's TMEM or exits while the other may still
  // arrive on its barriers or read its shared memory.
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Few rows (a decode step, a short prompt): bound by the bytes of W and, below
// that, by latency, so one short pipeline per CTA and no persistent walk.
//
// A cluster of `split` CTAs owns 128 rows of W and at most 64 activation rows
// (dense: a block of rows; grouped: the live slots of one block of one
// expert); its CTAs take equal ranges of K, so that a narrow W still streams
// through most SMs.  W comes through a TMA ring.  Behind this library's own
// quantisation pass it starts before griddepcontrol.wait: that pass lets its
// dependents in only once all work before it is complete, W's last writer
// included ([16 x 4096] -> 14336: 13.5 us, behind the wait 14.6).  Other
// kernels before it may have written W.  The activation comes
//   kTiles   by TMA through the same ring, its scales written once for the
//            CTA's whole range (dense MXFP8 rows);
//   kQuant   from 16-bit rows, quantised here with the rule of qdq_mxfp8 into
//            codes resident for the CTA's range (a handful of rows: one
//            launch instead of two);
//   kCopy    from MXFP8 rows by token index, resident likewise (grouped).
// The partial sums meet in distributed shared memory: each CTA adds the
// cluster's partials of its share of the W rows, always in rank order.
//
//   warp 0      TMA producer
//   warp 1      MMA issuer (M = 128, N = rows rounded up to 16, K = 32)
//   warps 2-9   activation fill in batches of 4 x 256 chunks of 8 elements,
//               one barrier a batch, then the epilogue
// ---------------------------------------------------------------------------
enum { kTiles = 0, kQuant = 1, kCopy = 2 };
constexpr int F_FILL = 256;
constexpr int F_THREADS = 64 + F_FILL;
constexpr int F_CHUNKS = TK / 8;          // 8-element chunks of a stage's row
constexpr int F_UNROLL = 4, F_BATCH = F_UNROLL * F_FILL;
constexpr int F_RING_MAX = 13, F_BATCH_MAX = 32;
constexpr int F_ROWS = 64;                // activation rows of an item at the most
constexpr int F_FILL_MAX = 96 * 1024;     // resident activation bytes of a CTA
constexpr uint32_t F_TMEM = 128, F_SFW = 64, F_SFA = 68;

struct __align__(8) FBars {
  uint64_t full[F_RING_MAX];
  uint64_t empty[F_RING_MAX];
  uint64_t ready[F_BATCH_MAX];  // the batch's groups (kTiles: all scales) are in shared memory
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort;
  int live;                     // grouped: live slots of the block
  int slot[F_ROWS];             // and their numbers
};

struct FewArgs {
  const void* a;               // 16-bit rows (kQuant) or codes (kCopy)
  int64_t lda;                 // elements / bytes
  const uint8_t* sfa;
  int64_t lds;
  const uint8_t* sfw;
  int64_t sf_per_expert;
  const void* bias;
  void* c;
  int64_t ldc;
  const int32_t* sorted_ids;
  const int32_t* expert_ids;
  const int32_t* num_post_padded;
  const float* topk_w;
  int M, N, K, kchunks;        // M: dense rows, grouped slots
  int rows, n_pad;             // rows of an item (grouped: block size), rounded up to 16
  int top_k, num_experts;
  int split, kt_per, ring;     // CTAs of a cluster, K-128 stages per CTA, stages in the ring
  int early;                   // W is complete before griddepcontrol.wait
  float zero;
  int* status;
};

template <int kDtype, bool kGrouped, int kAct>
__global__ void __launch_bounds__(F_THREADS, 1)
mxf8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                     const __grid_constant__ FewArgs p) {
  using O = Out16<kDtype>;
  using T = typename O::T;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // ring (W codes, kTiles: activation codes; the partial sums once the MMAs are done) | resident codes |
  // W scales | activation scales | barriers
  const int tile_a = p.n_pad * TK;  // a stage's activation codes
  const int stage_bytes = T_W + (kAct == kTiles ? tile_a : 0);
  uint8_t* s_act = smem + p.ring * stage_bytes;
  uint8_t* s_sfw = s_act + (kAct == kTiles ? 0 : p.kt_per * tile_a);
  uint8_t* s_sfa = s_sfw + p.ring * 512;
  FBars* bars = reinterpret_cast<FBars*>(s_sfa + p.kt_per * 512);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split;
  const int item = static_cast<int>(blockIdx.x) / p.split;
  const int n_tiles = (p.N + TM - 1) / TM;
  // dense: the row blocks of one W tile side by side, so that they share it in L2
  const int num_m = kGrouped ? 1 : (p.M + p.rows - 1) / p.rows;
  const int n_tile = kGrouped ? item % n_tiles : item / num_m;
  const int blk = kGrouped ? item / n_tiles : item - n_tile * num_m;
  const int row0 = blk * p.rows;  // first row, or first sorted position
  const int num_kt = (p.K + TK - 1) / TK;
  const int kt0 = rank * p.kt_per, nkt = max(0, min(p.kt_per, num_kt - kt0));

  int expert = 0;
  if (kGrouped) {
    pdl_wait();  // the routing may come from the kernel before
    expert = __ldcg(p.expert_ids + blk);
    // the whole cluster shares the block, so it leaves as one
    if (row0 >= __ldcg(p.num_post_padded) || expert < 0 || expert >= p.num_experts) return;
  }
  const int w_row = expert * p.N + n_tile * TM;
  const uint8_t* sfw = p.sfw + expert * p.sf_per_expert + (static_cast<int64_t>(n_tile) * p.kchunks + kt0) * 512;
  auto issue_w = [&](int kt, int s) {
    mbar_arrive_expect_tx(&bars->full[s], stage_bytes + 512);
    tma_load_2d(smem + s * stage_bytes, &tmap_w, (kt0 + kt) * TK, w_row, &bars->full[s]);
    bulk_load(s_sfw + s * 512, sfw + static_cast<int64_t>(kt) * 512, 512, &bars->full[s]);
  };
  auto issue_a = [&](int kt, int s) {
    if (kAct == kTiles)
      tma_load_2d(smem + s * stage_bytes + T_W, &tmap_a, (kt0 + kt) * TK, row0, &bars->full[s]);
  };
  const int pre = min(p.ring, nkt);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int i = 0; i < F_BATCH_MAX; ++i) mbar_init(&bars->ready[i], F_FILL);
    mbar_init(&bars->acc_full, 1);
    bars->abort = 0;
    fence_barrier_init();
    if (!kGrouped && !p.early) pdl_wait();
    for (int kt = 0; kt < pre; ++kt) issue_w(kt, kt);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, F_TMEM);
    tmem_relinquish();
    // Only now may the next kernel start: let in before this CTA's
    // tcgen05.alloc, it could hold the tensor memory that this one waits for.
    pdl_launch_dependents();
  }
  if (kGrouped && warp == 2) {  // the block's live slots, in order
    int n = 0;
    for (int r = lane; r < F_ROWS; r += 32) {
      const int s = r < p.rows ? __ldcg(p.sorted_ids + row0 + r) : -1;
      const bool ok = s >= 0 && s < p.M;
      const unsigned bal = __ballot_sync(0xffffffffu, ok);
      if (ok) bars->slot[n + __popc(bal & ((1u << lane) - 1u))] = s;
      n += __popc(bal);
    }
    if (lane == 0) bars->live = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);  // uniform
  const int rows = kGrouped ? bars->live : min(p.rows, p.M - row0);

  if (warp == 0) {
    // ---------------- producer (the whole warp walks, one lane issues)
    const bool leader = elect_one();
    if (kAct == kTiles) {
      pdl_wait();
      if (leader)
        for (int kt = 0; kt < pre; ++kt) issue_a(kt, kt);
    }
    int issued = pre;
    Cursor at;  // the second lap refills a slot once the first lap's MMAs have completed
    bool ok = true;
    for (int kt = pre; kt < nkt; ++kt, at.next(p.ring)) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[at.slot], at.phase, p.status, 0x701));
      if (!ok) break;
      if (leader) {
        issue_w(kt, at.slot);
        issue_a(kt, at.slot);
      }
      ++issued;
    }
    if (!ok) bars->abort = 1;
    for (int kt = max(0, issued - p.ring); kt < issued; ++kt)
      mbar_wait(&bars->full[kt % p.ring], (kt / p.ring) & 1, p.status, 0x702);
  } else if (warp == 1) {
    // ---------------- MMA issuer
    const bool leader = elect_one();
    const uint32_t idesc = idesc_mxf8(TM, (max(rows, 1) + 15) / 16 * 16);
    bool ok = true;
    int batches = 0, covered = 0;  // batches seen complete, and the chunks in them
    Cursor at;
    const uint64_t dw0 = smem_desc_sw128(smem), da0 = smem_desc_sw128(kAct == kTiles ? smem + T_W : s_act);
    const uint64_t dsw0 = smem_desc_sf(s_sfw), dsa0 = smem_desc_sf(s_sfa);
    auto stage = [&](int kt, int s) {
      tmem_cp_sf(tmem + F_SFW, dsw0 + (s * 512 >> 4));
      tmem_cp_sf(tmem + F_SFA, dsa0 + (kt * 512 >> 4));
      const uint64_t dw = dw0 + (s * stage_bytes >> 4);
      const uint64_t da = da0 + ((kAct == kTiles ? s * stage_bytes : kt * tile_a) >> 4);
#pragma unroll
      for (uint32_t kk = 0; kk < 4; ++kk)
        mma_mxf8(tmem, dw + 2 * kk, da + 2 * kk, idesc_with_sf_ids(idesc, kk, kk), (tmem + F_SFW) | (kk << 30),
                 (tmem + F_SFA) | (kk << 30), (kt | kk) != 0);
      tc_commit(&bars->empty[s]);
    };
    for (int kt = 0; kt < nkt;) {
      const int need = kAct == kTiles ? 1 : (kt + 1) * F_CHUNKS * rows;
      for (; ok && covered < need; covered += F_BATCH) ok = mbar_wait(&bars->ready[batches++], 0, p.status, 0x703);
      // four, two or one stage, as many as are full: the loop around them costs as much as two stages' issue
      const int more = min(nkt - kt, kAct == kTiles ? 4 : (covered - need) / max(1, F_CHUNKS * rows) + 1);
      Cursor c[4] = {at, at, at, at};
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        c[i] = c[i - 1];
        c[i].next(p.ring);
      }
      int n = 1;
      if (ok && more >= 4 && p.ring >= 4 &&
          __all_sync(0xffffffffu, mbar_test4(&bars->full[c[0].slot], c[0].phase, &bars->full[c[1].slot], c[1].phase,
                                             &bars->full[c[2].slot], c[2].phase, &bars->full[c[3].slot], c[3].phase)))
        n = 4;
      else if (ok && more >= 2 && p.ring >= 2 &&
               __all_sync(0xffffffffu, mbar_test2(&bars->full[c[0].slot], c[0].phase, &bars->full[c[1].slot], c[1].phase)))
        n = 2;
      else
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->full[c[0].slot], c[0].phase, p.status, 0x704));
      if (!ok) break;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) stage(kt + i, c[i].slot);
      }
      at = n == 4 ? c[3] : n == 2 ? c[1] : c[0];
      at.next(p.ring);
      kt += n;
    }
    if (!ok) bars->abort = 1;
    if (leader) tc_commit(&bars->acc_full);  // also on abort: the epilogue waits for the issued MMAs
  } else if (kAct == kTiles) {
    // ---------------- activation scales: a row's four bytes per stage, neighbouring lanes along the row (with
    // neighbouring lanes down the rows, the SMs' reads of the same few lines queued for 3 us)
    pdl_wait();
    const int words = nkt * rows;
    const uint32_t tail = scale_mask(p.K, num_kt - 1);
    for (int i0 = threadIdx.x - 64; i0 < words; i0 += 2 * F_FILL) {
      uint32_t v[2];
      int at[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = i0 + u * F_FILL, r = i / nkt, kt = i - r * nkt;
        at[u] = kt * 512 + (r & 31) * 16 + (r >> 5) * 4;
        if (i < words) v[u] = __ldcg(reinterpret_cast<const uint32_t*>(p.sfa + (row0 + r) * p.lds + (kt0 + kt) * 4));
        if (kt0 + kt + 1 == num_kt) v[u] &= tail;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (i0 + u * F_FILL < words) *reinterpret_cast<uint32_t*>(s_sfa + at[u]) = v[u];
    }
    fence_proxy_async_smem();
    mbar_arrive(&bars->ready[0]);
  } else {
    // ---------------- activation fill: chunk j (8 elements) of a stage's row, four neighbouring lanes a scale group
    if (!kGrouped) pdl_wait();
    const int chunks = nkt * F_CHUNKS * rows, per_stage = F_CHUNKS * rows;
    int batch = 0;
    for (int i0 = threadIdx.x - 64; i0 < (chunks + F_FILL - 1) / F_FILL * F_FILL; i0 += F_BATCH, ++batch) {
      uint4 v[F_UNROLL];
      uint32_t sb[F_UNROLL];
#pragma unroll
      for (int u = 0; u < F_UNROLL; ++u) {
        const int i = i0 + u * F_FILL, kt = i / per_stage, j = i - kt * per_stage, r = j / F_CHUNKS, c = j % F_CHUNKS;
        const int k = (kt0 + kt) * TK + c * 8;  // element of K; behind K: zero codes with scale 2^-127
        v[u] = make_uint4(0, 0, 0, 0);
        sb[u] = 0;
        if (i < chunks && k < p.K) {
          const int64_t tok = kGrouped ? bars->slot[r] / p.top_k : row0 + r;
          if (kAct == kQuant) {
            v[u] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.a) + tok * p.lda + k));
          } else {
            const uint2 w = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.a) + tok * p.lda + k));
            v[u].x = w.x;
            v[u].y = w.y;
            sb[u] = __ldcg(p.sfa + tok * p.lds + (k >> 5));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < F_UNROLL; ++u) {
        const int i = i0 + u * F_FILL, kt = i / per_stage, j = i - kt * per_stage, r = j / F_CHUNKS, c = j % F_CHUNKS;
        uint2 code = make_uint2(v[u].x, v[u].y);
        if (kAct == kQuant) {
          uint32_t amax = absmax8(v[u]);  // the lanes of a group walk together
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const int e = mx8_exp<kDtype>(amax);
          sb[u] = static_cast<uint32_t>(e);
          code = chunk_codes<kDtype>(v[u], e, p.zero);
        }
        if (i < chunks) {
          // 128-byte swizzle: 16-byte chunk h of row r sits at chunk h ^ (r % 8)
          *reinterpret_cast<uint2*>(s_act + kt * tile_a + r * TK + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8) = code;
          if ((c & 3) == 0) s_sfa[kt * 512 + (r & 31) * 16 + (r >> 5) * 4 + (c >> 2)] = static_cast<uint8_t>(sb[u]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&bars->ready[batch]);
    }
  }

  // ---------------- epilogue (warps 2-9): TMEM lanes = W rows, columns = activation rows.  The sums go through
  // shared memory, so that one short loop stores them in whole lines (an unrolled store per column cost 1.4 us of
  // instruction fetches).
  float* part = reinterpret_cast<float*>(smem);
  bool ok = true;
  if (warp >= 2) {
    const int q = warp & 3, half = (warp - 2) >> 2;
    ok = mbar_wait(&bars->acc_full, 0, p.status, 0x705);
    ok = __all_sync(0xffffffffu, ok && !*(volatile int*)&bars->abort);
    tc_fence_after();
    for (int c = 16 * half; c < rows; c += 32) {
      uint32_t acc[16];
      tmem_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, acc);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < rows) part[(c + i) * TM + q * 32 + lane] = nkt > 0 ? __uint_as_float(acc[i]) : 0.f;
    }
  }
  __syncwarp();
  if (p.split > 1) cluster_sync();  // every CTA's partials are in its shared memory
  else __syncthreads();
  if (warp >= 2 && ok) {
    const float* mine = part;
    auto add_up = [&](auto split_c) {  // split_c partials of each sum, 16 loads in flight a thread
      constexpr int kSplit = decltype(split_c)::value, kU = kSplit == 1 ? 8 : 16 / kSplit;
      // thread: one of this CTA's W rows, every `step`-th activation row
      constexpr int kShare = TM / kSplit, step = F_FILL / kShare;
      const int t = threadIdx.x - 64, row = rank * kShare + t % kShare, n = n_tile * TM + row;
      if (n >= p.N) return;
      T* C = static_cast<T*>(p.c) + n;
      const float bias = (!kGrouped && p.bias != nullptr) ? O::load(static_cast<const T*>(p.bias) + n) : 0.f;
#pragma unroll 1
      for (int r0 = t / kShare; r0 < rows; r0 += step * kU) {
        float x[kU][kSplit];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int c = 0; c < kSplit; ++c) {
            const float* from = mine + min(r0 + u * step, rows - 1) * TM + row;
            if (kSplit == 1) x[u][c] = *from;
            else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[u][c]) : "r"(cluster_addr(from, c)));
          }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int r = r0 + u * step;
          if (r >= rows) break;
          float v = x[u][0];
#pragma unroll
          for (int c = 1; c < kSplit; ++c) v += x[u][c];
          const int64_t s = kGrouped ? bars->slot[r] : row0 + r;
          if (kGrouped) v *= p.topk_w != nullptr ? __ldcg(p.topk_w + s) : 1.0f;
          else v += bias;
          C[s * p.ldc] = O::one(v);
        }
      }
    };
    if (p.split == 1) add_up(std::integral_constant<int, 1>());
    else if (p.split == 2) add_up(std::integral_constant<int, 2>());
    else if (p.split == 4) add_up(std::integral_constant<int, 4>());
    else add_up(std::integral_constant<int, 8>());
  }
  if (p.split > 1) {
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its partials
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, F_TMEM);
  }
}

// ---------------------------------------------------------------------------
// Segments of the grouped product: runs of consecutive live blocks that name
// the same expert, cut into at most nbmax blocks.  One CTA; blocks are walked
// in chunks of the CTA's size with carries, entries come out in order.
// ---------------------------------------------------------------------------
// Threads of the pass's CTAs.  Copying MXFP8 rows, three CTAs of 512 stand on an SM where one of 1024 did (calls in us,
// 512 and 1024 threads in turn: 64 tokens, 4 of 128 experts of 5760 x 2880 282.9 and 286.1, 4096 tokens 458 and 464; 911
// tokens, 2 of 4 of 390 x 224 8.4 and 9.2; 4096, 4 of 32 of 256 x 2880 36.4 and 37.9; one of eight shapes the other way,
// 2048 tokens, 2 of 8 of 512 x 8192 36.4 and 35.6); quantising, 1024 are faster (4096 tokens of K = 4096: 40.7, with 512
// 43.3).
constexpr int SEG_THREADS = 1024;
__host__ __device__ constexpr int prepare_threads(bool raw) { return raw ? SEG_THREADS : SEG_THREADS / 2; }

__device__ void build_segments(const int32_t* __restrict__ expert_ids, const int32_t* __restrict__ sorted_ids, int live,
                               int bs, int num_experts, int n_slots, int nbmax, int32_t* seg_tab) {
  __shared__ int s_start[32], s_count[32];
  __shared__ int s_expert[1 + SEG_THREADS + P_NT_MAX];  // the chunk's, the block's before it and nbmax behind it
  const int t = threadIdx.x, lane = t & 31, wid = t >> 5, nw = blockDim.x >> 5;
  int carry_start = -1, carry_count = 0;
  for (int base = 0; base < live; base += blockDim.x) {
    const int b = base + t;
    for (int i = t; i < 1 + static_cast<int>(blockDim.x) + P_NT_MAX; i += blockDim.x) {
      const int at = base - 1 + i;
      s_expert[i] = at >= 0 && at < live ? __ldcg(expert_ids + at) : -1;
    }
    __syncthreads();
    const int e = s_expert[1 + t];
    const bool valid = e >= 0 && e < num_experts;
    const bool first = valid && (b == 0 || s_expert[t] != e);
    int start = first ? b : -1;  // the first block of b's run: a running maximum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, start, o);
      if (lane >= o) start = max(start, v);
    }
    if (lane == 31) s_start[wid] = start;
    __syncthreads();
    for (int w = 0; w < wid; ++w) start = max(start, s_start[w]);
    start = max(start, carry_start);
    int last = carry_start;
    for (int w = 0; w < nw; ++w) last = max(last, s_start[w]);
    const bool seg = valid && (b - start) % nbmax == 0;
    const unsigned bal = __ballot_sync(0xffffffffu, seg);
    if (lane == 0) s_count[wid] = __popc(bal);
    __syncthreads();
    int at = carry_count + __popc(bal & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < wid) at += s_count[w];
      all += s_count[w];
    }
    if (seg) {
      int nb = 1;
      while (nb < nbmax && s_expert[1 + t + nb] == e) ++nb;  // nbmax <= P_NT_MAX
      reinterpret_cast<int4*>(seg_tab + 4)[at] = make_int4(b * bs, nb * bs, e, 0);
    }
    carry_start = last;
    carry_count += all;
    __syncthreads();
  }
  if (t == 0) seg_tab[0] = carry_count;
  // Padding at a segment's end costs MMAs and loads in steps of 16 rows: cut it, a warp four segments at a time, so
  // that their loads overlap.
  if (bs > 16) {
    constexpr int kU = 4;
    for (int i0 = wid * kU; i0 < carry_count; i0 += nw * kU) {
      int4 e[kU];
      int s[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        e[u] = i0 + u < carry_count ? reinterpret_cast<int4*>(seg_tab + 4)[i0 + u] : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int r = e[u].y - 1 - lane;
        s[u] = r >= 0 ? __ldcg(sorted_ids + e[u].x + r) : -1;
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        int rows = e[u].y;
        while (rows > 0) {
          const unsigned live_rows = __ballot_sync(0xffffffffu, s[u] >= 0 && s[u] < n_slots);
          if (live_rows != 0) {
            rows -= __ffs(live_rows) - 1;
            break;
          }
          rows = max(0, rows - 32);
          const int r = rows - 1 - lane;
          s[u] = r >= 0 ? __ldcg(sorted_ids + e[u].x + r) : -1;
        }
        if (lane == 0 && i0 + u < carry_count) seg_tab[4 + 4 * (i0 + u) + 1] = rows;
      }
    }
  }
}

// The pass before the grouped product: block 0 builds the segments, the others
// lay the routed rows out in sorted order, 2^wpr_log warps a row with four
// 16-byte loads in flight each, quantising 16-bit rows (kRaw) or copying MXFP8
// rows.  Positions that no live slot fills keep what the workspace held: their
// columns of the accumulators are dropped.  (Gathering the rows in the product
// instead, by 4-row TMA gathers, took 65 cycles a gather, 3100 a stage of 192
// rows against 600 with boxes of sorted rows.)
template <int kDtype, bool kRaw>
__global__ void __launch_bounds__(prepare_threads(kRaw))
mxf8_moe_prepare_kernel(const uint8_t* __restrict__ a, int64_t lda_bytes, const uint8_t* __restrict__ a_scales,
                        int64_t lds, const int32_t* __restrict__ sorted_ids, const int32_t* __restrict__ expert_ids,
                        const int32_t* __restrict__ num_post_padded, int bs, int num_blocks, int num_experts,
                        int nbmax, int top_k, int n_slots, int K, uint8_t* __restrict__ codes,
                        uint8_t* __restrict__ scales, int64_t ldso, int32_t* seg_tab, int wpr_log, float zero) {
  pdl_launch_dependents();
  pdl_wait();
  const int npp = __ldcg(num_post_padded);
  const int live = npp <= 0 ? 0 : min(num_blocks, (npp - 1) / bs + 1);
  if (blockIdx.x == 0) {
    build_segments(expert_ids, sorted_ids, live, bs, num_experts, n_slots, nbmax, seg_tab);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rpc = prepare_threads(kRaw) / 32 >> wpr_log;
  const int part = warp & ((1 << wpr_log) - 1);
  const int64_t positions = static_cast<int64_t>(live) * bs;
  const int gpr = K / 32;
  for (int64_t pos = static_cast<int64_t>(blockIdx.x - 1) * rpc + (warp >> wpr_log); pos < positions;
       pos += static_cast<int64_t>(gridDim.x - 1) * rpc) {
    const int s = __ldcg(sorted_ids + pos);
    if (s < 0 || s >= n_slots) continue;
    const uint4* src = reinterpret_cast<const uint4*>(a + static_cast<int64_t>(s / top_k) * lda_bytes);
    uint8_t* dst = codes + pos * K;
    const int chunks = (kRaw ? 4 : 2) * gpr;  // 16-byte chunks: 8 elements, four lanes a group; or 16 codes
    if (!kRaw) {
      const uint4* from = reinterpret_cast<const uint4*>(a_scales + static_cast<int64_t>(s / top_k) * lds);
      for (int c = part * 32 + lane; c < ldso / 16; c += 32 << wpr_log)
        reinterpret_cast<uint4*>(scales + pos * ldso)[c] = __ldcg(from + c);
    }
    for (int c0 = part * 128; c0 < chunks; c0 += 128 << wpr_log) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + 32 * u + lane;
        v[u] = c < chunks ? __ldcg(src + c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + 32 * u + lane;
        if (kRaw) {
          uint32_t amax = absmax8(v[u]);
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const int e = mx8_exp<kDtype>(amax);
          if (c < chunks) {
            *reinterpret_cast<uint2*>(dst + 8 * c) = chunk_codes<kDtype>(v[u], e, zero);
            if ((c & 3) == 0) scales[pos * ldso + (c >> 2)] = static_cast<uint8_t>(e);
          }
        } else if (c < chunks) {
          reinterpret_cast<uint4*>(dst)[c] = v[u];
        }
      }
    }
  }
}

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
bool off(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

template <typename... P, typename... A>
int launch_pdl(const char* who, void (*fn)(P...), int64_t grid, int threads, size_t smem, cudaStream_t s, int cluster,
               A... args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...);
  if (e != cudaSuccess) return fail(QDQ_ERR_CUDA, "%s: launch: %s", who, cudaGetErrorString(e));
  return check_launch(who);
}

template <typename F>
int allow_smem(const char* who, F fn, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e != cudaSuccess) return fail(QDQ_ERR_CUDA, "%s: smem attribute: %s", who, cudaGetErrorString(e));
    done[dev] = true;
  }
  return QDQ_OK;
}

template <int kDtype, bool kGrouped>
int launch_gemm(const char* who, const CUtensorMap& tw, const CUtensorMap& ta, const CUtensorMap& tsf, const GemmArgs& p,
                bool pair, int64_t items, cudaStream_t s) {
  if (pair) {
    static bool done[64] = {false};
    if (int st = allow_smem(who, &mxf8_pair_kernel<kDtype, kGrouped>, done)) return st;
    const int tok_rows = (p.nt / 2 + p.box - 1) / p.box * p.box;
    const int64_t pairs = std::min<int64_t>(items, device_sm_count() / 2);
    return launch_pdl(who, &mxf8_pair_kernel<kDtype, kGrouped>, 2 * pairs, T_THREADS, p_smem(tok_rows), s, 2, tw, ta, tsf, p);
  }
  static bool done[64] = {false};
  if (int st = allow_smem(who, &mxf8_gemm_kernel<kDtype, kGrouped>, done)) return st;
  return launch_pdl(who, &mxf8_gemm_kernel<kDtype, kGrouped>, std::min<int64_t>(items, device_sm_count()), T_THREADS,
                    t_smem(p.nt), s, 1, tw, ta, p);
}

// How a few-rows launch splits: `split` CTAs of a cluster share an item's K so
// that the items fill the SMs; split 0: the launch does not fit.  With more
// items than SMs (grouped) a CTA takes half of an SM's shared memory, so that
// two run side by side instead of in turn (4 of 128 experts, 5760 x 2880, 180
// items: 22.2 -> 17.5 us; with items below that, split CTAs two to an SM were
// no faster).
struct FewPlan {
  int split, kt_per, ring;
  size_t smem;
};
FewPlan few_plan(int64_t items, int rows, int64_t K, int act) {
  FewPlan f = {0, 0, 0, 0};
  const int num_kt = static_cast<int>((K + TK - 1) / TK), n_pad = (rows + 15) / 16 * 16;
  int split = 1;
  while (split < 8 && items * split * 2 <= device_sm_count() && num_kt >= split * 4) split *= 2;
  f.kt_per = (num_kt + split - 1) / split;
  const int64_t resident = static_cast<int64_t>(f.kt_per) * ((act == kTiles ? 0 : n_pad * TK) + 512);
  if (resident > F_FILL_MAX || (act != kTiles && f.kt_per * F_CHUNKS * rows > F_BATCH_MAX * F_BATCH)) return f;
  const int stage = T_W + (act == kTiles ? n_pad * TK : 0);
  const int most = items > device_sm_count() ? kSmemMax / 2 - 1024 : kSmemMax;  // 1 KB of each CTA's is the system's
  const int room = (most - 1024 - static_cast<int>(sizeof(FBars)) - static_cast<int>(resident)) / (stage + 512);
  // the ring also holds the partial sums, 512 bytes an activation row
  f.ring = std::max(std::min(std::min(room, F_RING_MAX), f.kt_per), (n_pad * TM * 4 + stage - 1) / stage);
  if (f.ring > room) return f;
  f.smem = 1024 + sizeof(FBars) + resident + static_cast<size_t>(f.ring) * (stage + 512);
  f.split = split;
  return f;
}

template <int kDtype, bool kGrouped, int kAct>
int launch_few(const char* who, const CUtensorMap& tw, const CUtensorMap& ta, const FewArgs& p, int64_t items,
               size_t smem, cudaStream_t s) {
  static bool done[64] = {false};
  if (int st = allow_smem(who, &mxf8_few_rows_kernel<kDtype, kGrouped, kAct>, done)) return st;
  return launch_pdl(who, &mxf8_few_rows_kernel<kDtype, kGrouped, kAct>, items * p.split, F_THREADS, smem, s, p.split, tw,
                    ta, p);
}

template <bool kGrouped, int kAct>
int run_few(const char* who, const CUtensorMap& tw, const CUtensorMap& ta, FewArgs& p, const FewPlan& f,
            int64_t items, int dtype, cudaStream_t s) {
  p.split = f.split;
  p.kt_per = f.kt_per;
  p.ring = f.ring;
  p.n_pad = (p.rows + 15) / 16 * 16;
  p.zero = 0.0f;  // +0.0 as an operand the compiler cannot fold (see mx8_scaled)
  return dtype == QDQ_DTYPE_FP16 ? launch_few<QDQ_DTYPE_FP16, kGrouped, kAct>(who, tw, ta, p, items, f.smem, s)
                                 : launch_few<QDQ_DTYPE_BF16, kGrouped, kAct>(who, tw, ta, p, items, f.smem, s);
}

// Which tiled kernel a dense product takes, and its rows per item.  The cycles
// of a K-128 stage are the largest of its MMAs' (2 per activation row), its
// operand bytes at 80 a cycle and its issue (300, pairs 430), plus 80; the
// launch takes as many stages as the busiest SM has items.  Against the best
// of five forced choices the rule's was within 6 % on 14 shapes, e.g.
// [4096 x 4096 -> 14336] pairs of 240 rows 181 us, single CTAs of 192 rows 213,
// and at the clock that a second of such calls settles at 208 and 252; [4096 x
// 1024 -> 512] single CTAs of 128 rows 8.2 us, pairs 10.2.
//
// Grouped: `segments(nt)` estimates the segments at nt rows per item from what
// the host knows, `rows` the rows of an average one.  Where every expert has one
// segment (`experts` of them) its weights come from memory, which gives an SM no
// stage in less than 700 cycles.  Both kernels then take the same time but for
// starts, tails and idle halves of pairs, and pairs that cost up to 6 % more
// stages are taken where their own stage is shorter (192 rows an item; pairs and
// single CTAs at the settled clock: 512 tokens, 8 experts of 14336 x 4096 102.6
// and 112.8 us; 4096 tokens, 128 experts of 2880 x 2880 248 and 272, of 5760 x
// 2880 457 and 510) or an SM has 16 items or more (128 experts of 5760 x 2880, 32
// tokens 219.9 and 226.9, 64 tokens 283 and 296; of 2880 x 2880, 128 tokens 165
// and 170.4; with 7 items, 16 tokens, 8 experts of 14336 x 4096, 82.6 and 79.3).
struct TilePlan {
  bool pair;
  int nt;
};
template <typename Segments>
TilePlan tile_plan(int64_t rows, int64_t blocks, int64_t experts, Segments segments) {
  TilePlan best = {false, 0};
  double least = 0, stage = 0;
  const int64_t sms = device_sm_count();
  for (int pair = 0; pair < 2; ++pair) {
    for (int nt = 16; nt <= (pair ? P_NT_MAX : NT_MAX); nt += 16) {
      const int64_t segs = segments(nt);
      if (segs <= 0) continue;
      const int64_t items = segs * (pair ? (blocks + 1) / 2 : blocks), units = pair ? sms / 2 : sms;
      const int64_t waves = (items + units - 1) / units;
      const double used = static_cast<double>(std::min<int64_t>(nt, rows));
      const double bytes = T_W + used * TK * (pair ? 0.5 : 1.0);
      const double own = std::max(std::max(2.0 * used, bytes / 80.0), pair ? 430.0 : 300.0) + 80.0;
      const bool streams = segs == experts;
      const double cost = static_cast<double>(waves) * std::max(own, streams ? 700.0 : 0.0);
      const bool liked = pair && !best.pair && streams && (own < stage || waves >= 16);
      if (best.nt == 0 || cost < (liked ? 1.06 : 1.0) * least) {
        best = {pair != 0, nt};
        least = cost;
        stage = own;
      }
    }
  }
  return best;
}

// The neighbouring n that C, rows of `ldc` elements of 16 bits, takes in one store.
int store_width(const void* c, int64_t ldc, int64_t N) {
  if (N % 8 == 0 && ldc % 8 == 0 && !off(c, 16)) return 8;
  return N % 2 == 0 && ldc % 2 == 0 && !off(c, 4) ? 2 : 1;
}

int check_product(const char* who, int dtype, int64_t M, int64_t N, int64_t K) {
  if (dtype != QDQ_DTYPE_BF16 && dtype != QDQ_DTYPE_FP16)
    return fail(QDQ_ERR_INVALID_ARG, "%s: dtype must be bf16 (0) or fp16 (1)", who);
  if (M < 0 || N < 0 || K < 0) return fail(QDQ_ERR_INVALID_ARG, "%s: negative shape", who);
  if (K % 32 != 0) return fail(QDQ_ERR_UNSUPPORTED, "%s: K=%lld must be a multiple of 32", who, (long long)K);
  if (M >= (1ll << 30) || N >= (1ll << 30) || K >= (1ll << 30))
    return fail(QDQ_ERR_UNSUPPORTED, "%s: dimension too large", who);
  if (K == 0 && M > 0 && N > 0) return fail(QDQ_ERR_UNSUPPORTED, "%s: K == 0", who);
  return QDQ_OK;
}

}  // namespace
}  // namespace qdqb200

using namespace qdqb200;

namespace qdqb200 {
namespace {

// The few-rows launch of a dense product from MXFP8 rows (raw == false) or
// 16-bit rows; false where the tiled kernel takes it.
bool dense_few(const char* who, const void* a, int64_t lda, const void* a_scales, int64_t lds, bool raw, bool early,
               const void* w_codes, const void* w_sf_tiled, const void* bias, void* c, int64_t M, int64_t N, int64_t K,
               int64_t ldw, int64_t ldc, int dtype, cudaStream_t s, int* st) {
  const int64_t n_tiles = (N + TM - 1) / TM;
  const int rows = static_cast<int>(std::min<int64_t>(M, F_ROWS));
  const int64_t items = n_tiles * ((M + rows - 1) / rows);
  if (items > device_sm_count()) return false;
  const FewPlan f = few_plan(items, rows, K, raw ? kQuant : kTiles);
  // 16-bit rows are quantised in the kernel while a CTA's share is one batch of its fill
  if (f.split == 0 || (raw && (M > F_ROWS || f.kt_per * F_CHUNKS * M > F_BATCH))) return false;
  FewArgs p = {};
  p.a = a;
  p.lda = lda;
  p.sfa = static_cast<const uint8_t*>(a_scales);
  p.lds = lds;
  p.sfw = static_cast<const uint8_t*>(w_sf_tiled);
  p.bias = bias;
  p.c = c;
  p.ldc = ldc;
  p.M = static_cast<int>(M);
  p.rows = rows;
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.kchunks = static_cast<int>((K / 32 + 7) / 8 * 2);
  p.top_k = 1;
  p.early = early;
  p.status = device_status_ptr();
  CUtensorMap tw, ta = {};
  *st = p.status == nullptr ? QDQ_ERR_CUDA : make_tmap_u8_2d(&tw, w_codes, N, K, ldw, TK, TM, 128);
  if (*st == QDQ_OK && !raw) *st = make_tmap_u8_2d(&ta, a, M, K, lda, TK, (rows + 15) / 16 * 16, 128);
  if (*st == QDQ_OK)
    *st = raw ? run_few<false, kQuant>(who, tw, ta, p, f, items, dtype, s)
              : run_few<false, kTiles>(who, tw, ta, p, f, items, dtype, s);
  return true;
}

int check_dense(const char* who, const void* w_codes, const void* w_sf_tiled, const void* bias, const void* c,
                int64_t N, int64_t K, int64_t ldw, int64_t ldc) {
  if (!w_codes || !w_sf_tiled || !c) return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (ldw < K || ldc < N) return fail(QDQ_ERR_INVALID_ARG, "%s: leading dimension too small", who);
  if (off(w_codes, 16) || ldw % 16 || off(w_sf_tiled, 16) || off(c, 2) || off(bias, 2))
    return fail(QDQ_ERR_ALIGNMENT, "%s: codes and scales must be 16-byte aligned", who);
  return QDQ_OK;
}

// fp8_gemm_mxf8; `early`: the launch before it is this library's quantisation pass.
int product_of_rows(const char* who, bool early, const void* a_codes, const void* a_scales, int64_t lda, int64_t lds,
                    const void* w_codes, const void* w_sf_tiled, const void* bias, void* c, int64_t M, int64_t N,
                    int64_t K, int64_t ldw, int64_t ldc, int out_dtype, void* stream) {
  if (int st = check_product(who, out_dtype, M, N, K)) return st;
  if (M == 0 || N == 0) return QDQ_OK;
  if (int st = check_dense(who, w_codes, w_sf_tiled, bias, c, N, K, ldw, ldc)) return st;
  if (!a_codes || !a_scales) return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (lda < K || lds < qdq_mxfp8_scale_stride(K))
    return fail(QDQ_ERR_INVALID_ARG, "%s: leading dimension too small", who);
  if (off(a_codes, 16) || lda % 16 || off(a_scales, 16) || lds % 16)
    return fail(QDQ_ERR_ALIGNMENT, "%s: codes and scales must be 16-byte aligned", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int few = QDQ_OK;
  if (dense_few(who, a_codes, lda, a_scales, lds, false, early, w_codes, w_sf_tiled, bias, c, M, N, K, ldw, ldc, out_dtype, s,
                &few))
    return few;
  int* status = device_status_ptr();
  if (status == nullptr) return QDQ_ERR_CUDA;
  GemmArgs p = {};
  p.sfw = static_cast<const uint8_t*>(w_sf_tiled);
  p.sfa = static_cast<const uint8_t*>(a_scales);
  p.lds = lds;
  p.bias = bias;
  p.c = c;
  p.ldc = ldc;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.kchunks = static_cast<int>((K / 32 + 7) / 8 * 2);
  p.a_rows = p.M;
  p.wide = store_width(c, ldc, N);
  const int64_t blocks = (N + TM - 1) / TM;
  const TilePlan plan = tile_plan(M, blocks, 0, [&](int nt) { return (M + nt - 1) / nt; });
  p.nt = plan.nt;
  p.box = plan.pair ? plan.nt / 2 : plan.nt;  // one tile's rows in one box
  p.status = status;
  CUtensorMap tw, ta, tsf = {};
  if (int st = make_tmap_u8_2d(&tw, w_codes, N, K, ldw, TK, TM, 128)) return st;
  if (int st = make_tmap_u8_2d(&ta, a_codes, M, K, lda, TK, p.box, 128)) return st;
  if (plan.pair)
    if (int st = make_tmap_u32_2d(&tsf, w_sf_tiled, blocks * p.kchunks, 128, 512, 128, 4)) return st;
  const int64_t items = ((M + p.nt - 1) / p.nt) * (plan.pair ? (blocks + 1) / 2 : blocks);
  if (items >= (1ll << 30)) return fail(QDQ_ERR_UNSUPPORTED, "%s: too many tiles", who);
  return out_dtype == QDQ_DTYPE_FP16 ? launch_gemm<QDQ_DTYPE_FP16, false>(who, tw, ta, tsf, p, plan.pair, items, s)
                                     : launch_gemm<QDQ_DTYPE_BF16, false>(who, tw, ta, tsf, p, plan.pair, items, s);
}

}  // namespace
}  // namespace qdqb200

extern "C" int fp8_gemm_mxf8(const void* a_codes, const void* a_scales, int64_t lda, int64_t lds,
                             const void* w_codes, const void* w_sf_tiled, const void* bias, void* c, int64_t M,
                             int64_t N, int64_t K, int64_t ldw, int64_t ldc, int out_dtype, void* stream) {
  return product_of_rows("fp8_gemm_mxf8", false, a_codes, a_scales, lda, lds, w_codes, w_sf_tiled, bias, c, M, N, K,
                         ldw, ldc, out_dtype, stream);
}

extern "C" int64_t fp8_linear_workspace_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  return up256(M * K) + up256(M * qdq_mxfp8_scale_stride(K));
}

extern "C" int fp8_linear_mxf8(const void* a, int64_t lda, int dtype, const void* w_codes, const void* w_sf_tiled,
                               const void* bias, void* c, int64_t M, int64_t N, int64_t K, int64_t ldw, int64_t ldc,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "fp8_linear_mxf8";
  if (int st = check_product(who, dtype, M, N, K)) return st;
  if (M == 0 || N == 0) return QDQ_OK;
  if (!a) return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if (int st = check_dense(who, w_codes, w_sf_tiled, bias, c, N, K, ldw, ldc)) return st;
  if (lda < K) return fail(QDQ_ERR_INVALID_ARG, "%s: leading dimension too small", who);
  if (off(a, 16) || lda % 8) return fail(QDQ_ERR_ALIGNMENT, "%s: rows of a must be 16-byte aligned", who);
  if (workspace == nullptr || off(workspace, 256) || workspace_bytes < fp8_linear_workspace_bytes(M, K))
    return fail(QDQ_ERR_INVALID_ARG, "%s: workspace missing, unaligned or smaller than fp8_linear_workspace_bytes()",
                who);
  int few = QDQ_OK;
  if (dense_few(who, a, lda, nullptr, 0, true, false, w_codes, w_sf_tiled, bias, c, M, N, K, ldw, ldc, dtype,
                static_cast<cudaStream_t>(stream), &few))
    return few;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + up256(M * K);
  const int64_t lds = qdq_mxfp8_scale_stride(K);
  // K % 32 == 0, so the codes' rows are 16-byte aligned at stride K
  if (int st = qdq_mxfp8_rows(a, codes, scales, M, K, lda, K, lds, dtype, stream)) return st;
  return product_of_rows(who, true, codes, scales, K, lds, w_codes, w_sf_tiled, bias, c, M, N, K, ldw, ldc, dtype,
                         stream);
}

extern "C" int64_t fp8_moe_workspace_bytes(int64_t size_m, int64_t num_sorted, int moe_block_size, int64_t K) {
  if (size_m <= 0 || num_sorted <= 0 || moe_block_size <= 0 || K <= 0) return 0;
  const int64_t row = qdq_mxfp8_scale_stride(K);
  return up256(16 * (1 + num_sorted / moe_block_size)) + up256(num_sorted * K) + up256(num_sorted * row) +
         up256(size_m * K) + up256(size_m * row);
}

extern "C" int fp8_moe_mxf8(const void* a, int64_t lda, const void* a_codes, const void* a_scales, int64_t ldac,
                            int64_t lds, int dtype, const void* w_codes, const void* w_sf_tiled, int64_t num_experts,
                            const int32_t* sorted_token_ids, const int32_t* expert_ids,
                            const int32_t* num_tokens_post_padded, const float* topk_weights, int64_t num_sorted,
                            int moe_block_size, int top_k, int mul_topk_weights, void* c, int64_t ldc,
                            int64_t size_m, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* who = "fp8_moe_mxf8";
  if (int st = check_product(who, dtype, size_m, N, K)) return st;
  if (num_sorted < 0 || num_experts < 0) return fail(QDQ_ERR_INVALID_ARG, "%s: negative size", who);
  if (moe_block_size < 1 || moe_block_size > 64)
    return fail(QDQ_ERR_UNSUPPORTED, "%s: moe_block_size must be in [1, 64] (got %d)", who, moe_block_size);
  if (top_k < 1) return fail(QDQ_ERR_INVALID_ARG, "%s: top_k must be >= 1", who);
  if (size_m == 0 || N == 0 || num_sorted == 0 || num_experts == 0) return QDQ_OK;
  if ((!a && (!a_codes || !a_scales)) || !w_codes || !w_sf_tiled || !sorted_token_ids || !expert_ids ||
      !num_tokens_post_padded || !c || (mul_topk_weights && !topk_weights))
    return fail(QDQ_ERR_INVALID_ARG, "%s: null pointer", who);
  if ((a ? lda < K : ldac < K || lds < qdq_mxfp8_scale_stride(K)) || ldc < N)
    return fail(QDQ_ERR_INVALID_ARG, "%s: leading dimension too small", who);
  if ((a ? off(a, 16) || lda % 8 : off(a_codes, 16) || ldac % 16 || off(a_scales, 16) || lds % 16) || off(w_codes, 16) ||
      off(w_sf_tiled, 16) || off(c, 2))
    return fail(QDQ_ERR_ALIGNMENT, "%s: codes and scales must be 16-byte aligned", who);
  if (num_experts >= (1ll << 31) / N || size_m >= (1ll << 30) / top_k || num_sorted >= (1ll << 30))
    return fail(QDQ_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (workspace == nullptr || off(workspace, 256) ||
      workspace_bytes < fp8_moe_workspace_bytes(size_m, num_sorted, moe_block_size, K))
    return fail(QDQ_ERR_INVALID_ARG, "%s: workspace missing, unaligned or smaller than fp8_moe_workspace_bytes()", who);
  const int64_t num_blocks = num_sorted / moe_block_size;
  if (num_blocks == 0) return QDQ_OK;
  const int64_t n_tiles = (N + TM - 1) / TM;
  if (num_blocks * n_tiles >= (1ll << 30)) return fail(QDQ_ERR_UNSUPPORTED, "%s: too many tiles", who);
  int* status = device_status_ptr();
  if (status == nullptr) return QDQ_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap tw, ta;
  if (int st = make_tmap_u8_2d(&tw, w_codes, num_experts * N, K, K, TK, TM, 128)) return st;
  const int64_t n_slots = size_m * top_k;
  // A decode step of few blocks: one launch without quantisation pass or segments, an item per block.
  if (num_blocks * n_tiles <= 2 * device_sm_count()) {
    const FewPlan f = few_plan(num_blocks * n_tiles, moe_block_size, K, a ? kQuant : kCopy);
    if (f.split != 0) {
      FewArgs p = {};
      p.a = a ? a : a_codes;
      p.lda = a ? lda : ldac;
      p.sfa = static_cast<const uint8_t*>(a_scales);
      p.lds = lds;
      p.sfw = static_cast<const uint8_t*>(w_sf_tiled);
      p.sf_per_expert = qdq_sf_tiled_bytes(N, K);
      p.c = c;
      p.ldc = ldc;
      p.sorted_ids = sorted_token_ids;
      p.expert_ids = expert_ids;
      p.num_post_padded = num_tokens_post_padded;
      p.topk_w = mul_topk_weights ? topk_weights : nullptr;
      p.M = static_cast<int>(n_slots);
      p.N = static_cast<int>(N);
      p.K = static_cast<int>(K);
      p.kchunks = static_cast<int>((K / 32 + 7) / 8 * 2);
      p.rows = moe_block_size;
      p.top_k = top_k;
      p.num_experts = static_cast<int>(num_experts);
      p.status = status;
      ta = {};
      return a ? run_few<true, kQuant>(who, tw, ta, p, f, num_blocks * n_tiles, dtype, s)
               : run_few<true, kCopy>(who, tw, ta, p, f, num_blocks * n_tiles, dtype, s);
    }
  }
  int32_t* seg_tab = static_cast<int32_t*>(workspace);
  uint8_t* codes = static_cast<uint8_t*>(workspace) + up256(16 * (1 + num_blocks));
  uint8_t* scales = codes + up256(num_sorted * K);
  const int64_t ldso = qdq_mxfp8_scale_stride(K);
  // 16-bit rows that several slots read are quantised once, by a pass of their own, where it spares the pass below 2^23
  // elements (4096 tokens, 4 of 32 experts, K = 2880: 60 -> 49 us a call; 1024 tokens, 8 of 32, K = 2048: 31 -> 27.5;
  // 2048 tokens, 4 of 32, K = 1024, 6 M spared: no difference; 1024 tokens, 2 of 32, K = 2048, 2 M: 15.9 -> 17.3).
  bool raw = a != nullptr;
  if (raw && top_k > 1 && size_m * (top_k - 1) >= (1ll << 23) / K) {
    uint8_t* once = scales + up256(num_sorted * ldso);
    uint8_t* once_scales = once + up256(size_m * K);
    if (int st = qdq_mxfp8_rows(a, once, once_scales, size_m, K, lda, K, ldso, dtype, stream)) return st;
    raw = false;
    a_codes = once;
    a_scales = once_scales;
    ldac = K;
    lds = ldso;
  }
  GemmArgs p = {};
  // An average expert's rows in whole blocks, over as many experts as can be hit.  Few rows per item leave the shared
  // memory to more stages of W in flight; boxes leave a ragged segment few idle rows.
  const int64_t experts = std::min(num_experts, num_blocks);
  const int64_t average = ((num_sorted + experts - 1) / experts + moe_block_size - 1) / moe_block_size * moe_block_size;
  const TilePlan plan = tile_plan(average, n_tiles, experts, [&](int nt) {
    const int64_t rows = nt / moe_block_size * moe_block_size;
    return rows == 0 ? int64_t(0) : experts * ((average + rows - 1) / rows);
  });
  const bool pair = plan.pair;
  p.nt = plan.nt;
  const int held = pair ? p.nt / 2 : p.nt;  // rows in one CTA's shared memory
  p.box = held > 96 ? 64 : held > 16 ? 32 : held > 8 ? 16 : 8;
  if (!pair) p.nt = std::min(NT_MAX, (p.nt + p.box - 1) / p.box * p.box);
  const int nbmax = p.nt / moe_block_size;
  {
    // Several warps a row (128 chunks each) while all of them are resident at once.
    const int threads = prepare_threads(raw), warps = threads / 32, per_sm = raw ? 1 : 3;
    int wpr_log = 0;
    while ((2 << wpr_log) <= warps && (128ll << wpr_log) < K / (raw ? 8 : 16) &&
           (num_sorted << wpr_log) <= static_cast<int64_t>(per_sm) * warps * device_sm_count())
      ++wpr_log;
    const int64_t rpc = warps >> wpr_log;
    const int64_t grid = 1 + std::min<int64_t>((num_sorted + rpc - 1) / rpc, std::max(2, per_sm) * device_sm_count());
    auto* fn = !raw ? &mxf8_moe_prepare_kernel<QDQ_DTYPE_BF16, false>
               : dtype == QDQ_DTYPE_FP16 ? &mxf8_moe_prepare_kernel<QDQ_DTYPE_FP16, true>
                                         : &mxf8_moe_prepare_kernel<QDQ_DTYPE_BF16, true>;
    if (int st = launch_pdl(who, fn, grid, threads, 0, s, 1, static_cast<const uint8_t*>(raw ? a : a_codes),
                            raw ? lda * 2 : ldac, static_cast<const uint8_t*>(a_scales), lds, sorted_token_ids,
                            expert_ids, num_tokens_post_padded, moe_block_size, num_blocks, num_experts, nbmax, top_k,
                            n_slots, K, codes, scales, ldso, seg_tab, wpr_log, 0.0f))
      return st;
  }
  p.sfw = static_cast<const uint8_t*>(w_sf_tiled);
  p.sf_per_expert = qdq_sf_tiled_bytes(N, K);
  p.sfa = scales;
  p.lds = ldso;
  p.a_rows = static_cast<int>(num_sorted);
  p.c = c;
  p.ldc = ldc;
  p.seg_tab = seg_tab;
  p.wide = store_width(c, ldc, N);
  p.sorted_ids = sorted_token_ids;
  p.topk_w = mul_topk_weights ? topk_weights : nullptr;
  p.M = static_cast<int>(n_slots);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.kchunks = static_cast<int>((K / 32 + 7) / 8 * 2);
  p.num_blocks = static_cast<int>(num_blocks);
  p.num_experts = static_cast<int>(num_experts);
  p.status = status;
  if (int st = make_tmap_u8_2d(&ta, codes, num_sorted, K, K, TK, p.box, 128)) return st;
  CUtensorMap tsf = {};
  if (pair)
    if (int st = make_tmap_u32_2d(&tsf, w_sf_tiled, num_experts * (p.sf_per_expert / 512), 128, 512, 128, 4)) return st;
  const int64_t items = num_blocks * (pair ? (n_tiles + 1) / 2 : n_tiles);
  return dtype == QDQ_DTYPE_FP16 ? launch_gemm<QDQ_DTYPE_FP16, true>(who, tw, ta, tsf, p, pair, items, s)
                                 : launch_gemm<QDQ_DTYPE_BF16, true>(who, tw, ta, tsf, p, pair, items, s);
}
