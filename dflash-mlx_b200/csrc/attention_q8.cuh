// What the two forms of the attention over an 8-bit cache share (attention_q8.cu,
// attention_q8_tc.cu): arguments, code conversion and row limits.
#pragma once
#include "kv_q8.cuh"

namespace dfl {

// A row's exponentials e_j = 2^(x_j - M) are taken relative to a base M that follows the maximum of x_j plus the
// exponent of vs_j (q8_exponent) over the keys it has seen, that is the largest weight e_j vs_j, so that the weights
// fit fp16 whichever keys have the large scores and whichever the large scales. A key's e_j is then at most 2^14 over
// its scale's exponent: that counts as Q8_EXP_MIN at least (V scales below 2^-104 are the first to lose bits), and the
// sums of e_j are kept in units of 2^16, so that with V scales up to 2^90 neither they nor the weights leave fp32's
// normal range, over 2^20 keys and more.
// Two bases may so lie more than 2^126 apart with sums that count alike (a key of weight 1/2 and V scale 2^-90, then
// one of 2^80): sums are rescaled by the root of the factor twice, at every place where they are. For weights and
// accumulators a factor below fp32's range may be 0.
// In a block of keys whose exponents lie within Q8_NEAR of one another the maximum of the x_j plus the largest
// exponent stands for that maximum, at most Q8_NEAR above it. Rows that see the whole of such a block take it, all
// others the exact one: a rule on the row's own keys. (Exact in every block, 64 x 16 rows of 32 heads take 127 us in
// place of 116, 1024 prompt rows 149 in place of 131.)
constexpr int Q8_EXP_MIN = -104;
constexpr int Q8_NEAR = 4;
constexpr float Q8_SUM_UNIT = 1.f / 65536.f;
// The base starts Q8_BASE below that maximum and is raised when it lags by Q8_LAZY (log2), so weights stay below 2^15
// and the largest is 1 at least, 2^4 where the V scales are alike. (8 and 6 would give it four bits more, and rescale
// oftener: 64 x 16 rows 118 -> 126 us, 8 gated blocks at head_dim 256 50 -> 55.)
constexpr float Q8_BASE = 4.f, Q8_LAZY = 10.f;

// What a row's products q' . Kc ks are multiplied by to be x_j: the softmax scale and the power of two that q' was
// scaled by. At least 2^-126, with which the scores of such a row are all alike: 0 times a masked key's -inf is NaN.
__device__ __forceinline__ float q8_row_factor(float scale_log2, int sh) {
  return fmaxf(scale_log2 * __uint_as_float((uint32_t)(127 - sh) << 23), 1.17549435e-38f);
}

// floor(log2 |v|) of a V scale, at least Q8_EXP_MIN; Q8_EXP_MIN too for infinities and NaN, whose exponent field
// becomes 0 when 1 is added
__device__ __forceinline__ int q8_exponent(float v) {
  return max((int)(((__float_as_uint(v) + 0x00800000u) >> 23) & 0xffu) - 128, Q8_EXP_MIN);
}

// 2^x, results below the normal range flushed to zero (fp16 weights and their sum lose nothing)
__device__ __forceinline__ float q8_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

struct AttnQ8Args {
  const __nv_bfloat16* q;  // [M][Hq][hd]
  Q8Cache c;
  const int* pos;
  const int* row_seq;
  const int* kv_len;
  float* part_o;    // [chunks][M][Hq][hd]
  float2* part_ml;  // [chunks][M][Hq]: (M, sum)
  __nv_bfloat16* out;
  long long ldo;
  const __nv_bfloat16* gate;
  long long ldg;
  int gate_hs;
  int M, Hq, G, causal, max_kv, n_chunks, key_chunk;
  int run_rows;   // rows per run
  int runs;       // runs of the call
  int ranked;     // the launch takes the runs with the most keys first
  int tile_toks;  // tokens per tile
  int run_tiles;  // tiles per run
  float scale_log2;  // |softmax scale| * log2(e); 1 when the scale is 0
  float q_sign;      // sign of the softmax scale (0 when it is 0): folded into q
  int* err;
};

__device__ __forceinline__ uint32_t hsub2_u32(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four codes b0..b3 to two half2: (b0, b1), (b2, b3) with PAIRED (K: consecutive dims) or
// (b0, b2), (b1, b3) without (V: the same dim of two keys).
template <bool E4M3, bool PAIRED>
__device__ __forceinline__ void q8_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    if (!PAIRED) w = __byte_perm(w, 0, 0x3120);
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // fp16 0x6400 | u is 1024 + u; the biased byte u = c + 128
    w ^= 0x80808080u;
    lo = hsub2_u32(__byte_perm(w, 0x64646464u, PAIRED ? 0x4140 : 0x4240), 0x64806480u);
    hi = hsub2_u32(__byte_perm(w, 0x64646464u, PAIRED ? 0x4342 : 0x4341), 0x64806480u);
  }
}

// keys row m sees: clamped to what the cache and the call allow (an excess sets the error word). kv_len from L2: the
// merge kernel asks before it waits, when this SM's L1 may still hold the entry as an earlier kernel read it.
__device__ __forceinline__ int q8_row_limit(const AttnQ8Args& a, int m, int p, int seq, int* err) {
  const long long lim = a.causal ? (long long)p + 1 : __ldcg(a.kv_len + seq);
  const int most = min(a.max_kv, a.c.cap);
  if (lim > most) q8_error(err, Q8_ERR_POS);
  return lim > most ? most : lim < 0 ? 0 : (int)lim;
}

// Tile and kv head of a CTA: heads of a run side by side, runs in the launch's order. That order is by keys,
// most first (ties by index), where a.ranked: a long run started last would leave the other SMs idle
// (64 runs of 512 to 4096 keys, tcgen05 form: 169 us in index order, 130 so, before later steps). Every CTA
// ranks the runs alike from their last rows' limits, a permutation whatever those are.
constexpr int Q8_RANK_RUNS = 256;
struct Q8Tile {
  int run, tile, kvh;
};
__device__ __forceinline__ Q8Tile q8_tile(const AttnQ8Args& a) {
  __shared__ int4 s_keys[Q8_RANK_RUNS / 4];
  __shared__ int s_run;
  Q8Tile t;
  const int id = blockIdx.x / a.c.Hkv;
  t.kvh = blockIdx.x - id * a.c.Hkv;
  t.run = id / a.run_tiles;
  t.tile = id - t.run * a.run_tiles;
  if (!a.ranked) return t;
  const int n4 = (a.runs + 3) & ~3;
  for (int r = threadIdx.x; r < n4; r += blockDim.x) {
    int key = -1;
    if (r < a.runs) {
      const int m = min((r + 1) * a.run_rows, a.M) - 1;
      key = a.pos[m];
      if (!a.causal && key >= 0) {
        const int seq = a.row_seq ? a.row_seq[m] : 0;
        key = seq >= 0 && seq < a.c.n_seqs ? a.kv_len[seq] : 0;
      }
      key = max(key, 0);
    }
    reinterpret_cast<int*>(s_keys)[r] = key;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < a.runs; r += blockDim.x) {
    const int key = reinterpret_cast<const int*>(s_keys)[r];
    int rank = 0;
    for (int j = 0; j < n4 / 4; ++j) {  // runs before r win ties; the padding (-1) never counts
      const int4 k = s_keys[j];
      rank += (k.x > key || (k.x == key && 4 * j < r)) + (k.y > key || (k.y == key && 4 * j + 1 < r)) +
              (k.z > key || (k.z == key && 4 * j + 2 < r)) + (k.w > key || (k.w == key && 4 * j + 3 < r));
    }
    if (rank == t.run) s_run = r;
  }
  __syncthreads();
  t.run = s_run;
  return t;
}

// The tcgen05 forms (attention_q8_tc.cu), tiles of 64 rows or, wide, of 256 (head_dim 256: 128): the chunk kernel alone.
int launch_attention_q8_tc(const AttnQ8Args& a, int hd, bool e4m3, int rows, int tiles, cudaStream_t st);

}  // namespace dfl
