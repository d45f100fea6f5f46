// Attention over the 8-bit K/V cache on the 5th-generation tensor cores (tcgen05, accumulators and
// softmax weights in TMEM), for long key chunks. Same work split, masks, scales and partial-result
// format as attn_q8_kernel (attention_q8.cu); same independence of a row from its tile.
//
// One CTA per (run tile, kv head, key chunk), in two shapes:
//  * tc: tiles of up to 64 (token, head) rows. The 128-row MMA tile holds them twice: copy 0 (TMEM lanes
//    0-63) takes keys 0-31 of every 64-key block, copy 1 (lanes 64-127) keys 32-63, so that all four softmax
//    warps have work; the copies are merged at the end. Two CTAs an SM (one at head_dim 256).
//  * wide, for prefill: a row once, and two groups of 128 rows and four softmax warps each that share the
//    converted tiles (256 rows; at head_dim 256, where TMEM holds one group, 128). One CTA an SM. 1024 rows of
//    32 heads of 128 at 4096 keys: 109 us, 0.55 PFLOP/s (tc: 175 us).
// Per block and group:
//   S = Q K^T      M = 128, N = 64, K = hd, both operands fp16 in shared memory
//   w = e vs       one thread per (row, copy), 32 (wide: 64) keys each; fp16, over S's own TMEM columns, the
//                  other copy's keys zero
//   O += w V       A = w from TMEM, B = V as [key][dim] in shared memory (MN-major), N = hd
// Four softmax and epilogue warps a group, then four that convert codes to fp16 tiles (two K, two V), the last
// issues the MMAs. The converters load codes straight into registers, one block ahead of the one they convert.
// What bounds it is the chain of these roles, not one unit (64 blocks of 16, 512 to 4096 keys: 119 us, 44 % of
// the copy rate; at 130 us leaving out the softmax arithmetic gave 108, the MMAs 113, the loads 122; issue slots
// are 46 % busy). A block's softmax takes about 1200 clocks, and the issuing thread, at 58 clocks an MMA, 80 a
// commit and 130 a wait even for a barrier that is complete, nearly as many: it has one wait and two commits a
// block (with a barrier for each tile: 130 instead of 124 us, wide 129 instead of 111). A CTA's start and end,
// 12000 clocks, are a chain of latencies too, with several rows side by side (one row after the other, and Q loaded
// behind the positions: 18000 clocks, 124 us).
// A row's exponent base M follows its largest weight (score plus exponent of the V scale) lazily: sums, weights and
// O are rescaled only when M would grow by more than 10 (log2), so weights stay below 2^15 in fp16, and those down to
// 2^-14 of the largest keep all their bits (attention_q8.cuh).
// Every wait is bounded (device error 350-359).
#include "attention_q8.cuh"
#include "tcgen05.cuh"

namespace dfl {

constexpr int QT_KB = 64;       // keys per block
constexpr int QT_SCALES = 4;    // scale ring: block i's are read until its weights are written

template <int HD, int CP, int SG>  // CP copies of the rows in each of SG softmax groups' 128-row MMA tiles
struct QtLayout {
  static constexpr int ROWS = 128 / CP * SG;  // (token, head) rows per tile
  static constexpr int CONV = 4 * SG, ISSUER = CONV + 4;  // first converter warp, the issuing warp
  static constexpr int THREADS = 32 * (ISSUER + 1);
  static constexpr int UNITS = HD / 64;  // 64-dim (128-byte) units of an fp16 row
  static constexpr int TILE = QT_KB * HD * 2;
  static constexpr int OFF_K = 0;               // 2 stages
  static constexpr int OFF_V = 2 * TILE;        // 2 stages
  static constexpr int OFF_Q = 4 * TILE;        // [group][units][128 rows][128 B]; the epilogue reuses K, V and Q for O
  static constexpr int OFF_S = OFF_Q + SG * 128 * HD * 2;  // [4][64]: K scales, V scales, V exponents
  static constexpr int OFF_E = OFF_S + QT_SCALES * 3 * QT_KB * 4;  // [4][2]: largest, smallest V exponent of 32 keys
  static constexpr int OFF_R = OFF_E + QT_SCALES * 16;             // row factor, limit, (M, l) of all copies, output weights
  static constexpr int OFF_BAR = OFF_R + ROWS * 8 + SG * 128 * 8 + ROWS * 16;
  static constexpr int N_BAR = 2 + SG * 2 * 3;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static constexpr int GCOLS = 128 + HD;  // a group's columns: S / weights 2 x 64, O hd
  static constexpr uint32_t COLS = SG * GCOLS > 256 ? 512 : 256;
  static_assert(SG * GCOLS <= 512, "TMEM columns");
  static_assert(OFF_S >= SG * 128 * HD * 4, "O of all copies fits the K, V and Q tiles");
};

__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tc_st16_nowait(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Bounded wait that sleeps in the barrier unit (1 ms a try) instead of spending issue slots
__device__ __forceinline__ bool qt_wait(uint64_t* bar, uint32_t parity, int site, int* err) {
  const uint32_t addr = smem_u32(bar);
  for (int n = 0; n < 2000; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(1000000u)
        : "memory");
    if (ok) return true;
  }
  q8_error(err, site);
  return false;
}

// 16-byte chunk c of row r of a [rows][128 B] 128-byte-swizzled unit
__device__ __forceinline__ uint32_t qt_sw(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// kind::f16, A = B = fp16, D = fp32, M = 128; B K-major (S) or MN-major (O)
__host__ __device__ constexpr uint32_t qt_idesc(int n, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

template <int HD, bool E4M3, int CP, int SG>
__global__ void __launch_bounds__((QtLayout<HD, CP, SG>::THREADS), HD == 256 || SG > 1 ? 1 : 2)
    attn_q8_tc_kernel(const __grid_constant__ AttnQ8Args a) {
  using L = QtLayout<HD, CP, SG>;
  constexpr int ROWS = L::ROWS, LANE_ROWS = ROWS / 32;
  constexpr int KT = QT_KB / CP;  // keys of a block that a softmax thread takes
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* s_sc = reinterpret_cast<float*>(smem + L::OFF_S);  // [ring][K, V, exponents of V][64]
  float2* s_ve = reinterpret_cast<float2*>(smem + L::OFF_E);  // [ring][half]
  float* s_rowf = reinterpret_cast<float*>(smem + L::OFF_R);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::OFF_R + ROWS * 8);  // [128 SG]
  float4* s_w = reinterpret_cast<float4*>(s_ml + SG * 128);  // [rows]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  // k_full: K of the first two blocks. s_full and pv_done (MMA commits) also give their block's K and V tiles
  // back to the converters. p_full: a block's weights written (and its scores consumed), and, for group 0, its V
  // and the K of two blocks on converted: the one barrier that the issuer waits for per block and group.
  uint64_t* k_full = bars;             // [2]
  uint64_t* s_full = bars + 2;         // [SG][2]
  uint64_t* p_full = s_full + SG * 2;  // [SG][2]
  uint64_t* pv_done = p_full + SG * 2; // [SG][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::N_BAR);
  __shared__ int s_tok_lim[ROWS], s_tok_ok[ROWS];
  __shared__ int s_row[ROWS];  // token * 16 + head in group of each tile row, -1 behind the last

  grid_dependency_wait();
  const Q8Tile at = q8_tile(a);
  const int run = at.run, tile = at.tile, kvh = at.kvh, chunk = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = run * a.run_rows + tile * a.tile_toks;
  const int ntok = min(min(a.tile_toks, a.run_rows - tile * a.tile_toks), a.M - m0);
  if (ntok <= 0) return;
  // the tile's rows, two, four or eight a lane (tiles of 64, 128, 256), by every warp alike: their positions and
  // sequences, the run's sequence (that of the first row with a position), limits
  int pos2[LANE_ROWS], sq2[LANE_ROWS], seq = 0;
  bool any = false;
#pragma unroll
  for (int k = 0; k < LANE_ROWS; ++k) {
    const int i = lane + 32 * k;
    pos2[k] = i < ntok ? a.pos[m0 + i] : -1;
    sq2[k] = i < ntok && a.row_seq ? a.row_seq[m0 + i] : 0;
  }
  const int n_rows = ntok * a.G, groups = SG == 1 || n_rows <= 128 ? 1 : SG;
  // The softmax warps' Q rows, on their way while positions and limits are looked up: raw, into the last copy's place
  // (hd / 16 lanes a row, 32 bytes each), where each thread later converts what it copied. Rolled loops here and
  // there: code that runs once a CTA comes from a cold instruction cache.
  constexpr int GR = 128 / CP, LPR = HD / 16, QPW = 32 / LPR;  // a group's rows, lanes a row, rows a warp
  const int ql = lane % LPR, qr = (warp & 3) * QPW + lane / LPR, g0 = (warp >> 2) * GR;
  unsigned char* q1 = smem + L::OFF_Q + (warp >> 2) * 128 * HD * 2 + (ql >> 2) * 16384 + (CP - 1) * GR * 128;
  if (warp < L::CONV) {
    const float inv_g = 1.f / (float)a.G;
#pragma unroll 1
    for (int r = qr; r < GR; r += 4 * QPW) {
      const bool ok = g0 + r < n_rows;
      const int tok = (int)(((float)(g0 + r) + 0.5f) * inv_g);  // (g0 + r) / G: at least 1 / 32 from an integer
      const __nv_bfloat16* q =
          ok ? a.q + ((long long)(m0 + tok) * a.Hq + kvh * a.G + (g0 + r - tok * a.G)) * HD + ql * 16 : a.q;
      const uint32_t d = smem_u32(q1) + qt_sw(r, (ql & 3) * 2);
      cp_async16(d, q, ok ? 16 : 0);
      cp_async16(d ^ 16, q + (ok ? 8 : 0), ok ? 16 : 0);
    }
    cp_async_commit();
  }
#pragma unroll
  for (int k = LANE_ROWS - 1; k >= 0; --k) {
    const unsigned v = __ballot_sync(0xffffffffu, pos2[k] >= 0);
    const int s = __shfl_sync(0xffffffffu, sq2[k], v ? __ffs(v) - 1 : 0);
    if (v) seq = s;
    any = any || v;
  }
  if (!any) {
    cp_async_wait<0>();
    return;
  }
  if (seq < 0 || seq >= a.c.n_seqs) {  // a row that names no sequence of the cache is left as it is
    if (threadIdx.x == 0) q8_error(a.err, Q8_ERR_SEQ);
    cp_async_wait<0>();
    return;
  }
  int lim_max = 0, lim_min = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < LANE_ROWS; ++k) {
    const int i = lane + 32 * k;
    const bool ok = pos2[k] >= 0 && sq2[k] == seq;
    if (warp == 0 && pos2[k] >= 0 && !ok) q8_error(a.err, Q8_ERR_SEQ);
    const int lim = ok ? q8_row_limit(a, m0 + i, pos2[k], seq, warp == 0 && chunk == 0 && kvh == 0 ? a.err : nullptr) : 0;
    if (warp == 0) {
      s_tok_lim[i] = lim;
      s_tok_ok[i] = ok;
    }
    lim_max = max(lim_max, lim);
    if (lim > 0) lim_min = min(lim_min, lim);
  }
  lim_max = __reduce_max_sync(0xffffffffu, lim_max);
  lim_min = __reduce_min_sync(0xffffffffu, lim_min);
  const int k_begin = chunk * a.key_chunk;
  if (k_begin >= lim_max && a.n_chunks > 1) {
    cp_async_wait<0>();
    return;
  }
  const int k_end = min(k_begin + a.key_chunk, lim_max);
  const int n_blocks = (max(k_end - k_begin, 0) + QT_KB - 1) / QT_KB;
  if (threadIdx.x == 32 * L::ISSUER) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 64);
      for (int g = 0; g < groups; ++g) {
        mbar_init(&s_full[2 * g + s], 1);
        mbar_init(&p_full[2 * g + s], CP * ((min(n_rows - g * 128, 128) + 31) / 32) * 32 + (g == 0 ? 128 : 0));
        mbar_init(&pv_done[2 * g + s], 1);
      }
    }
    fence_barrier_init();
  }
  for (int r = threadIdx.x; r < ROWS; r += L::THREADS) {
    const int tok = r / a.G;
    s_row[r] = tok < ntok ? tok * 16 + r - tok * a.G : -1;
  }
  __syncthreads();
  const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
  if (warp >= L::CONV && warp < L::ISSUER) {
    // ---------------- converters: two warps K, two V ----------------
    constexpr int NC = HD / 16;            // 16-code chunks per key
    constexpr int PER = QT_KB * NC / 64;   // chunks per thread and block
    const int ct = threadIdx.x & 63;
    const bool is_v = warp >= L::CONV + 2;
    const unsigned char* src = (is_v ? a.c.v : a.c.k) + kvh * a.c.head_stride;
    const float* ks_src = a.c.ks + kvh * a.c.s_head_stride + ct;
    const float* vs_src = a.c.vs + kvh * a.c.s_head_stride + ct;
    unsigned char* dst = smem + (is_v ? L::OFF_V : L::OFF_K);
    float* sdst = s_sc + ct;
    uint64_t* empty = (is_v ? pv_done : s_full) + 2 * (groups - 1);
    // A thread's chunk column c and rows r, r + STEP, ... Lane bits: two of the chunk, one of the row,
    // the rest of the chunk, the rest of the row: the eight lanes of a 16-byte store phase write two
    // rows' chunks of one unit, eight different bank groups. STEP is a multiple of 4; for head_dim 256
    // odd multiples flip the swizzle's third bit.
    constexpr int HI = NC / 4, STEP = 64 / NC;
    const int c = (ct & 3) | (((ct >> 3) & (HI - 1)) << 2);
    const int r = ((ct >> 2) & 1) | ((ct / (8 * HI)) << 1);
    const uint32_t dst0 = (uint32_t)(c >> 2) * (QT_KB * 128) + qt_sw(r, (c & 3) * 2);
    src += c * 16;
    // Codes and scale offsets of 32 blocks, one a lane, made together: a table lookup per block would
    // stand in front of the block's loads. A place that is refused is -1: its keys have scale 0.
    int win = 0;
    long long win_off = -1, win_soff = 0;
    auto window = [&](int i) {
      long long page = 0;
      int row = 0;
      win = i;
      win_off = -1;
      if (i + lane < n_blocks && q8_place(a.c, seq, k_begin + (i + lane) * QT_KB, warp == L::CONV ? a.err : nullptr, page, row)) {
        win_off = page * a.c.seq_stride + (long long)row * HD;
        win_soff = page * a.c.s_seq_stride + row;
      }
    };
    // block i's codes and scale offsets; its keys, 0 behind the last block
    auto where = [&](int i, long long& off, long long& soff) -> int {
      off = __shfl_sync(0xffffffffu, win_off, i - win);
      soff = __shfl_sync(0xffffffffu, win_soff, i - win);
      return off < 0 ? 0 : min(QT_KB, k_end - (k_begin + i * QT_KB));
    };
    uint4 b[PER];
    // The thread's chunks of a block of n keys at p: volatile, so that the loads are issued here, most of
    // a block's time ahead of their use. Rows behind the last key repeat it: their scores are masked,
    // their weights 0, and a code is a finite number.
    auto fetch = [&](const unsigned char* p, int n) {
      if (n == QT_KB) {
#pragma unroll
        for (int u = 0; u < PER; ++u)
          asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                       : "=r"(b[u].x), "=r"(b[u].y), "=r"(b[u].z), "=r"(b[u].w)
                       : "l"(p + (r + u * STEP) * HD));
      } else if (n > 0) {
#pragma unroll
        for (int u = 0; u < PER; ++u)
          asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                       : "=r"(b[u].x), "=r"(b[u].y), "=r"(b[u].z), "=r"(b[u].w)
                       : "l"(p + min(r + u * STEP, n - 1) * HD));
      } else {
#pragma unroll
        for (int u = 0; u < PER; ++u) b[u] = make_uint4(0, 0, 0, 0);
      }
    };
    long long off, soff;
    window(0);
    int n = where(0, off, soff);
    fetch(src + off, n);
    // both scales of a key come through the K warps: they are there when the block's scores are
    float ks = !is_v && ct < n ? __ldg(ks_src + soff) : 0.f, vs = !is_v && ct < n ? __ldg(vs_src + soff) : 0.f;
    const int n_turns = n_blocks + (is_v || n_blocks == 0 ? 0 : 2);  // K is two blocks ahead of the barrier it arrives on
    for (int i = 0; i < n_turns; ++i) {
      const int s = i & 1;
      if (i + 1 - win >= 32) window(i + 1);
      n = where(i + 1, off, soff);
      if (!qt_wait(&empty[s], ((i >> 1) & 1) ^ 1, 350, a.err)) break;
      if (i >= n_blocks) {
        mbar_arrive(i < 2 ? &k_full[s] : &p_full[s]);
        continue;
      }
      if (!is_v) {
        float* sd = sdst + (i & (QT_SCALES - 1)) * 3 * QT_KB;
        sd[0] = ks;
        sd[QT_KB] = vs;
        const int e = q8_exponent(vs);
        sd[2 * QT_KB] = (float)e;
        const int e_max = __reduce_max_sync(0xffffffffu, e), e_min = __reduce_min_sync(0xffffffffu, e);  // of 32 keys
        if (lane == 0) s_ve[(i & (QT_SCALES - 1)) * 2 + (ct >> 5)] = make_float2((float)e_max, (float)e_min);
      }
      unsigned char* d = dst + s * L::TILE + dst0;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        uint4 h0, h1;
        q8_to_half<E4M3, true>(b[u].x, h0.x, h0.y);
        q8_to_half<E4M3, true>(b[u].y, h0.z, h0.w);
        q8_to_half<E4M3, true>(b[u].z, h1.x, h1.y);
        q8_to_half<E4M3, true>(b[u].w, h1.z, h1.w);
        // the chunk's second half lies at its first's address with bit 4 flipped
        const uint32_t flip = STEP % 8 ? (u & 1) << 6 : 0;
        unsigned char* du = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(d) ^ flip) + u * STEP * 128;
        *reinterpret_cast<uint4*>(du) = h0;
        *reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(du) ^ 16) = h1;
      }
      fetch(src + off, n);
      if (!is_v) {
        ks = ct < n ? __ldg(ks_src + soff) : 0.f;
        vs = ct < n ? __ldg(vs_src + soff) : 0.f;
      }
      fence_proxy_async_smem();
      mbar_arrive(!is_v && i < 2 ? &k_full[s] : &p_full[s]);
    }
  } else if (warp == L::ISSUER) {
    // ---------------- MMA issuer ----------------
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "n"(L::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    tc_fence_before();
    asm volatile("bar.sync 2, %0;\n" ::"n"(SG * 128 + 32) : "memory");  // Q written, TMEM allocated
    tc_fence_after();
    grid_dependency_launch_dependents();  // not before the allocation: a dependent's must not come first
    const uint32_t tmem = *tmem_slot;  // a group's S / weights: columns 0-63, 64-127, O from 128 on
    // The whole warp walks the loop, so that descriptors stay in uniform registers; one lane issues.
    uint32_t elected;  // by elect.sync rather than by lane number: wide 106 -> 103 us
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(elected));
    const bool leader = elected != 0;
    const uint64_t qd = sw128_desc(smem_u32(smem + L::OFF_Q));
    const uint64_t kd0 = sw128_desc(smem_u32(smem + L::OFF_K));
    const uint64_t vd0 = sw128_mn_desc(smem_u32(smem + L::OFF_V), QT_KB * 128, 1024);
    auto qk = [&](int i, int g) {
      const int s = i & 1;
      const uint32_t ts = tmem + g * L::GCOLS + s * 64;
      const uint64_t qg = qd + g * (128 * HD * 2 >> 4), kd = kd0 + s * (L::TILE >> 4);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        tc_mma(ts, qg + (kk >> 2) * (16384 >> 4) + 2 * (kk & 3), kd + (kk >> 2) * (QT_KB * 128 >> 4) + 2 * (kk & 3),
               qt_idesc(QT_KB, false), kk > 0 ? 1u : 0u);
      tc_commit(&s_full[2 * g + s]);
    };
    auto pv = [&](int j, int g) {
      const int s = j & 1;
      const uint64_t vd = vd0 + s * (L::TILE >> 4);
      const uint32_t tw = tmem + g * L::GCOLS + s * 64, t_o = tmem + g * L::GCOLS + 128;
#pragma unroll
      for (int kk = 0; kk < QT_KB / 16; ++kk)
        tc_mma_ts(t_o, tw + kk * 8, vd + kk * (2048 >> 4), qt_idesc(HD, true), j > 0 || kk > 0 ? 1u : 0u);
      tc_commit(&pv_done[2 * g + s]);
    };
    bool ok = true;
    for (int i = 0; i < min(n_blocks, 2) && ok; ++i) {
      ok = qt_wait(&k_full[i], 0, 354, a.err);
      if (!ok) break;
      tc_fence_after();
      if (leader)
        for (int g = 0; g < groups; ++g) qk(i, g);
      __syncwarp();
    }
    // Behind a block's barrier nothing stands between its product and the scores of two blocks on, which overwrite
    // its weights (the tensor core takes them in order).
    for (int j = 0; j < n_blocks && ok; ++j) {
      const int s = j & 1, ph = (j >> 1) & 1;
      for (int g = 0; g < groups && ok; ++g) {
        ok = qt_wait(&p_full[2 * g + s], ph, 352, a.err);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          pv(j, g);
          if (j + 2 < n_blocks) qk(j + 2, g);
        }
        __syncwarp();
      }
    }
  } else {
    // ---------------- softmax: thread = (row, copy), four warps a group ----------------
    // Q rows to scaled fp16, CP times; a row's factor undoes its power of two. U rows of a warp side by side, as
    // each is a chain of shared-memory and shuffle latencies.
    {
      constexpr int TURNS = GR / (4 * QPW), U = TURNS < 4 ? TURNS : 4;
      cp_async_wait<0>();
#pragma unroll 1
      for (int r = qr; r < GR; r += 4 * QPW * U) {
        uint4* d0[U];
        uint32_t u[U][8], mx[U];
#pragma unroll
        for (int t = 0; t < U; ++t) {
          d0[t] = reinterpret_cast<uint4*>(q1 + qt_sw(r + t * 4 * QPW, (ql & 3) * 2));
          const uint4 n0 = *d0[t], n1 = *reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(d0[t]) ^ 16);
          u[t][0] = n0.x, u[t][1] = n0.y, u[t][2] = n0.z, u[t][3] = n0.w;
          u[t][4] = n1.x, u[t][5] = n1.y, u[t][6] = n1.z, u[t][7] = n1.w;
        }
        // magnitudes compare as integers; one that is not finite leaves the row unscaled
#pragma unroll
        for (int t = 0; t < U; ++t) {
          uint32_t m2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) m2[j] = __vmaxu2(u[t][j] & 0x7fff7fffu, u[t][j + 4] & 0x7fff7fffu);
          m2[0] = __vmaxu2(__vmaxu2(m2[0], m2[1]), __vmaxu2(m2[2], m2[3]));
          mx[t] = max(m2[0] << 16, m2[0] & 0xffff0000u);
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1)
#pragma unroll
          for (int t = 0; t < U; ++t) mx[t] = max(mx[t], __shfl_xor_sync(0xffffffffu, mx[t], o));
#pragma unroll
        for (int t = 0; t < U; ++t) {
          const int sh = mx[t] > 0 && mx[t] < 0x7f800000u ? min(14 - ((int)(mx[t] >> 23) - 127), 120) : 0;
          const float f = __uint_as_float((uint32_t)(sh + 127) << 23) * a.q_sign;
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const __half2 y =
                __floats2half2_rn(__uint_as_float(u[t][j] << 16) * f, __uint_as_float(u[t][j] & 0xffff0000u) * f);
            h[j] = *reinterpret_cast<const uint32_t*>(&y);
          }
          const uint4 h0 = make_uint4(h[0], h[1], h[2], h[3]), h1 = make_uint4(h[4], h[5], h[6], h[7]);
          uint4* d1 = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(d0[t]) ^ 16);
          *d0[t] = h0;
          *d1 = h1;
          if (CP == 2) {
            *(d0[t] - GR * 8) = h0;  // the first copy, 64 rows of 128 bytes before
            *(d1 - GR * 8) = h1;
          }
          if (ql == 0) s_rowf[g0 + r + t * 4 * QPW] = q8_row_factor(a.scale_log2, sh);
        }
      }
    }
    fence_proxy_async_smem();
    tc_fence_before();
    asm volatile("bar.sync 2, %0;\n" ::"n"(SG * 128 + 32) : "memory");
    tc_fence_after();
    const int grp = SG == 1 ? 0 : warp >> 2;
    s_full += 2 * grp;
    p_full += 2 * grp;
    const uint32_t tmem = *tmem_slot + grp * L::GCOLS, t_o = tmem + 128;
    const int row = threadIdx.x & (ROWS - 1), half = CP == 2 ? threadIdx.x >> 6 : 0;
    const int lim = s_row[row] < 0 ? 0 : s_tok_lim[s_row[row] >> 4];
    const float rowf = s_rowf[row];
    float m = -INFINITY, mu_used = -INFINITY;  // m: largest x_j + exponent of vs_j
    uint64_t l = 0;  // two partial sums
    bool ok = true;
    // a warp whose 32 rows all lie behind the tile's does nothing: what its lanes hold goes to its own
    // rows of O, which nobody reads
    const int my_blocks = (row & ~31) < n_rows ? n_blocks : 0;
    for (int i = 0; i < my_blocks && ok; ++i) {
      const int s = i & 1;
      const float* sc = s_sc + (i & (QT_SCALES - 1)) * 3 * QT_KB + half * 32;
      const int kb = k_begin + i * QT_KB + half * 32;
      ok = qt_wait(&s_full[s], (i >> 1) & 1, 356, a.err);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool full = kb + KT <= lim_min;
      uint64_t x[KT / 2];
#pragma unroll
      for (int k = 0; k < KT; k += 32) {
        float sv[32];
        tc_ld32(tmem + lane_base + (uint32_t)(s * 64 + half * 32 + k), sv);
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const ulonglong2 ks = *reinterpret_cast<const ulonglong2*>(sc + k + 2 * c);
          x[k / 2 + c] = q8_mul2(q8_pack(sv[2 * c], sv[2 * c + 1]), ks.x);
          x[k / 2 + c + 1] = q8_mul2(q8_pack(sv[2 * c + 2], sv[2 * c + 3]), ks.y);
        }
      }
      if (!full) {
#pragma unroll
        for (int c = 0; c < KT / 2; ++c) {
          const float2 y = q8_unpack(x[c]);
          x[c] = q8_pack(kb + 2 * c < lim ? y.x : -INFINITY, kb + 2 * c + 1 < lim ? y.y : -INFINITY);
        }
      }
      const uint64_t rf2 = q8_pack(rowf, rowf);
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int c = 0; c < KT / 2; c += 2) {
        const float2 y = q8_unpack(x[c]), z = q8_unpack(x[c + 1]);
        mx0 = fmaxf(fmaxf(mx0, y.x), y.y);
        mx1 = fmaxf(fmaxf(mx1, z.x), z.y);
      }
      float2 ve = s_ve[(i & (QT_SCALES - 1)) * 2 + half];
      if (CP == 1) {
        const float2 other = s_ve[(i & (QT_SCALES - 1)) * 2 + 1];
        ve = make_float2(fmaxf(ve.x, other.x), fminf(ve.y, other.y));
      }
      const bool near = ve.x - ve.y <= (float)Q8_NEAR;
      float mx = __fmaf_rn(fmaxf(mx0, mx1), rowf, ve.x);
      if (!full || !near) {
        mx0 = mx1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < KT / 2; c += 2) {
          const ulonglong2 ex = *reinterpret_cast<const ulonglong2*>(sc + 2 * QT_KB + 2 * c);
          const float2 y = q8_unpack(q8_fma2(x[c], rf2, ex.x)), z = q8_unpack(q8_fma2(x[c + 1], rf2, ex.y));
          mx0 = fmaxf(fmaxf(mx0, y.x), y.y);
          mx1 = fmaxf(fmaxf(mx1, z.x), z.y);
        }
        if (!near || kb + KT > lim) mx = fmaxf(mx0, mx1);
      }
      m = fmaxf(m, mx);
      const float M = m - Q8_BASE;
      const bool grow = M > mu_used + Q8_LAZY || (mu_used == -INFINITY && M > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {  // a factor of 1 is exact
        const float root = grow ? q8_exp2(0.5f * (mu_used - M)) : 1.f, fac = root * root;
        if (grow) mu_used = M;
        l = q8_mul2(q8_mul2(l, q8_pack(root, root)), q8_pack(root, root));
        if (i > 0) {
          ok = qt_wait(&pv_done[2 * grp + ((i - 1) & 1)], ((i - 1) >> 1) & 1, 357, a.err);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            float ov[16];
            tc_ld16(t_o + lane_base + (uint32_t)c, ov);
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] *= fac;
            tc_st16(t_o + lane_base + (uint32_t)c, ov);
          }
        }
      }
      const float mu = mu_used == -INFINITY ? 0.f : mu_used;
      const uint64_t mu2 = q8_pack(-mu, -mu), unit2 = q8_pack(Q8_SUM_UNIT, Q8_SUM_UNIT);
      const uint32_t t_w = tmem + lane_base + (uint32_t)(s * 64);
#pragma unroll
      for (int k = 0; k < KT; k += 32) {
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const ulonglong2 vs = *reinterpret_cast<const ulonglong2*>(sc + QT_KB + k + 2 * c);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const float2 y = q8_unpack(q8_fma2(x[k / 2 + c + d], rf2, mu2));
            const uint64_t e = q8_pack(q8_exp2(y.x), q8_exp2(y.y));
            l = q8_fma2(e, unit2, l);
            const float2 ww = q8_unpack(q8_mul2(e, d ? vs.y : vs.x));
            const __half2 h = __floats2half2_rn(ww.x, ww.y);
            w[c + d] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        if (!full) {  // 0 * scale of a key that is not seen may be NaN
#pragma unroll
          for (int c = 0; c < 16; ++c)
            w[c] &= (kb + k + 2 * c < lim ? 0xffffu : 0u) | (kb + k + 2 * c + 1 < lim ? 0xffff0000u : 0u);
        }
        tc_st16_nowait(t_w + half * 16 + k / 2, w);
      }
      if (CP == 2) {
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) w[c] = 0;
        tc_st16_nowait(t_w + (half ^ 1) * 16, w);
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }
    // ---- O of both copies through shared memory, then merged, row by row ----
    const int nb1 = n_blocks - 1;
    for (int g = 0; g < groups && n_blocks > 0; ++g)  // every group's: O goes where all read K, V and Q
      if (ok) ok = qt_wait(&pv_done[2 * g + (nb1 & 1)], (nb1 >> 1) & 1, 358, a.err);
    ok = __all_sync(0xffffffffu, ok);
    constexpr int CH = HD / 4;  // float4 chunks per row
    float4* s_o = reinterpret_cast<float4*>(smem);
    if (ok && my_blocks > 0) {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float ov[32];
        tc_ld32(t_o + lane_base + (uint32_t)c, ov);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s_o[threadIdx.x * CH + ((c / 4 + e) ^ (threadIdx.x & 7))] =
              make_float4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
      }
      tc_fence_before();
    }
    s_ml[threadIdx.x] = make_float2(mu_used, q8_unpack(l).x + q8_unpack(l).y);
    asm volatile("bar.sync 1, %0;\n" ::"n"(SG * 128) : "memory");
    // a thread a row: the copies' weights, the quotient where this chunk is the only one, and where it goes (over
    // the row factors, and the thread's own (M, l), read no more)
    long long* s_dst = reinterpret_cast<long long*>(s_rowf);
    long long* s_gate = reinterpret_cast<long long*>(s_ml);
    if (threadIdx.x < ROWS) {
      const int r = threadIdx.x, th = s_row[r], tok = th >> 4;
      const float2 x0 = s_ml[r], x1 = CP == 2 ? s_ml[r + ROWS] : make_float2(-INFINITY, 0.f);
      const float mm = fmaxf(x0.x, x1.x), mu = mm == -INFINITY ? 0.f : mm;
      const float r0 = q8_exp2(0.5f * (x0.x - mu)), r1 = q8_exp2(0.5f * (x1.x - mu)), w0 = r0 * r0, w1 = r1 * r1;
      const float den = r0 * x0.y * r0 + r1 * x1.y * r1;
      float inv = 1.f;
      long long dst = -1, gate = 0;  // where the row of the output (or of the partials) begins, and its gate's
      if (ok && th >= 0 && s_tok_ok[tok] && (a.n_chunks == 1 || lim > k_begin)) {
        const long long m = m0 + tok, head = kvh * a.G + (th & 15);
        if (a.n_chunks > 1) {
          const long long to = ((long long)chunk * a.M + m) * a.Hq + head;
          a.part_ml[to] = make_float2(mm, den);
          dst = to * HD;
        } else {
          inv = lim > 0 ? Q8_SUM_UNIT / den : 0.f;
          dst = m * a.ldo + head * HD;
          gate = m * a.ldg + head * a.gate_hs;
        }
      }
      s_w[r] = make_float4(w0, w1, lim > 0 ? 1.f : 0.f, inv);
      s_dst[r] = dst;
      s_gate[r] = gate;
    }
    asm volatile("bar.sync 1, %0;\n" ::"n"(SG * 128) : "memory");
    constexpr int RPW = CH >= 32 ? 1 : 32 / CH;  // rows a warp writes at a time
    constexpr int NR = 4, STEP = 4 * SG * RPW;   // times in flight, rows between them
    constexpr int NC = CH >= 32 ? CH / 32 : 1;   // float4s a lane has of a row
    const int c0 = lane % (32 / RPW);
    const bool wide_gate = (reinterpret_cast<uintptr_t>(a.gate) % 8 | a.ldg % 4 | a.gate_hs % 4) == 0;
#pragma unroll 1
    for (int r0 = warp * RPW + lane / (32 / RPW); r0 < n_rows; r0 += NR * STEP) {
      float4 y[NR][NC];
      float inv[NR];
      long long dst[NR];
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        const int r = min(r0 + u * STEP, ROWS - 1);
        const float4 w = s_w[r];
        inv[u] = w.w;
        dst[u] = r0 + u * STEP < n_rows ? s_dst[r] : -1;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int c = (c0 + 32 * k) ^ (r & 7);
          const float4 o0 = s_o[r * CH + c];
          float4 v = make_float4(w.x * o0.x, w.x * o0.y, w.x * o0.z, w.x * o0.w);
          if (CP == 2) {
            const float4 o1 = s_o[(r + ROWS) * CH + c];
            v = make_float4(v.x + w.y * o1.x, v.y + w.y * o1.y, v.z + w.y * o1.z, v.w + w.y * o1.w);
          }
          y[u][k] = w.z != 0.f ? v : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      if (a.n_chunks > 1) {
#pragma unroll
        for (int u = 0; u < NR; ++u)
#pragma unroll
          for (int k = 0; k < NC; ++k)
            if (dst[u] >= 0) *reinterpret_cast<float4*>(a.part_o + dst[u] + (c0 + 32 * k) * 4) = y[u][k];
        continue;
      }
      // The copies' sum first, then the quotient, as the merge kernel has it (its sum starts at +0, so that no zero
      // is negative): a row whose keys lie in the first chunk has the same bits in calls of one chunk and of several.
#pragma unroll
      for (int u = 0; u < NR; ++u)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          y[u][k].x = (y[u][k].x + 0.f) * inv[u];
          y[u][k].y = (y[u][k].y + 0.f) * inv[u];
          y[u][k].z = (y[u][k].z + 0.f) * inv[u];
          y[u][k].w = (y[u][k].w + 0.f) * inv[u];
        }
      if (a.gate) {
        uint2 g[NR][NC];
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          if (dst[u] < 0) continue;
          const __nv_bfloat16* gr = a.gate + s_gate[r0 + u * STEP] + c0 * 4;
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            if (wide_gate) {
              g[u][k] = *reinterpret_cast<const uint2*>(gr + 128 * k);
            } else {
              const unsigned short* gs = reinterpret_cast<const unsigned short*>(gr + 128 * k);
              g[u][k] = make_uint2(gs[0] | (uint32_t)gs[1] << 16, gs[2] | (uint32_t)gs[3] << 16);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < NR; ++u)
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            y[u][k].x /= 1.f + __expf(-__uint_as_float(g[u][k].x << 16));
            y[u][k].y /= 1.f + __expf(-__uint_as_float(g[u][k].x & 0xffff0000u));
            y[u][k].z /= 1.f + __expf(-__uint_as_float(g[u][k].y << 16));
            y[u][k].w /= 1.f + __expf(-__uint_as_float(g[u][k].y & 0xffff0000u));
          }
      }
#pragma unroll
      for (int u = 0; u < NR; ++u)
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (dst[u] >= 0)
            *reinterpret_cast<uint2*>(a.out + dst[u] + (c0 + 32 * k) * 4) =
                make_uint2(pack_bf16x2(y[u][k].x, y[u][k].y), pack_bf16x2(y[u][k].z, y[u][k].w));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == L::ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(*tmem_slot), "n"(L::COLS));
  }
}

template <int HD, bool E4M3, int CP, int SG>
static int launch_qt(const AttnQ8Args& a, int tiles, cudaStream_t st) {
  using L = QtLayout<HD, CP, SG>;
  static bool opted[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    if (cudaFuncSetAttribute(attn_q8_tc_kernel<HD, E4M3, CP, SG>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) !=
        cudaSuccess) {
      cudaGetLastError();
      set_error("dfl_attention_q8: cannot opt in to %d bytes of shared memory", L::SMEM);
      return DFL_ERR_UNSUPPORTED;
    }
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * a.c.Hkv, a.n_chunks);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_q8_tc_kernel<HD, E4M3, CP, SG>, a);
  if (e != cudaSuccess) {
    set_error("dfl_attention_q8: launch failed: %s", cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

template <int HD, bool E4M3>
static int launch_qt_rows(const AttnQ8Args& a, int rows, int tiles, cudaStream_t st) {
  return rows == 64 ? launch_qt<HD, E4M3, 2, 1>(a, tiles, st) : launch_qt<HD, E4M3, 1, HD == 256 ? 1 : 2>(a, tiles, st);
}

int launch_attention_q8_tc(const AttnQ8Args& a, int hd, bool e4m3, int rows, int tiles, cudaStream_t st) {
  switch (hd) {
    case 64: return e4m3 ? launch_qt_rows<64, true>(a, rows, tiles, st) : launch_qt_rows<64, false>(a, rows, tiles, st);
    case 128: return e4m3 ? launch_qt_rows<128, true>(a, rows, tiles, st) : launch_qt_rows<128, false>(a, rows, tiles, st);
    default: return e4m3 ? launch_qt_rows<256, true>(a, rows, tiles, st) : launch_qt_rows<256, false>(a, rows, tiles, st);
  }
}

}  // namespace dfl
