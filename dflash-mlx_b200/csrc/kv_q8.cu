// Writing and reading the 8-bit K/V cache.
//
//  * dfl_qkv_rope_append_q8 - per-head q/k RMSNorm, RoPE and the append that quantises each key
//                             and value row as it is written
//  * dfl_kv_read_q8         - cache rows back as bf16
//
// A row of hd values x is held as codes c and one fp32 scale s, x ~ c * s (int8: s = max|x| / 127;
// e4m3: max|x| / 448). Both kernels are bound by memory: per row the append reads the
// projection's (Hq + 2 Hkv) * hd bf16 values and writes Hq * hd bf16 and 2 Hkv (hd + 4) bytes.
#include "kv_q8.cuh"

namespace dfl {

int q8_cache(const dfl_kv_q8* c, const char* who, Q8Cache* out) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
    set_error("%s: null cache, codes or scales", who);
    return DFL_ERR_INVALID;
  }
  if (c->type != DFL_KV_INT8 && c->type != DFL_KV_E4M3) {
    set_error("%s: cache type %d is neither DFL_KV_INT8 nor DFL_KV_E4M3", who, c->type);
    return DFL_ERR_INVALID;
  }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    set_error("%s: head_dim %d not supported (64, 128, 256)", who, c->head_dim);
    return DFL_ERR_UNSUPPORTED;
  }
  if (c->n_kv_heads <= 0 || c->n_kv_heads > 65535 || c->n_seqs <= 0 || c->cap <= 0 || c->seq_stride < 0 ||
      c->head_stride < 0 || c->scale_seq_stride < 0 || c->scale_head_stride < 0) {
    set_error("%s: bad cache geometry (Hkv=%d n_seqs=%d cap=%d)", who, c->n_kv_heads, c->n_seqs, c->cap);
    return DFL_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 || c->seq_stride % 16 ||
      c->head_stride % 16) {
    set_error("%s: cache codes must be 16-byte aligned, with strides that are multiples of 16", who);
    return DFL_ERR_UNSUPPORTED;
  }
  int shift = 0;
  if (c->page_table) {
    if (c->page_size < 64 || (c->page_size & (c->page_size - 1)) || c->pt_stride <= 0 || c->n_pages <= 0) {
      set_error("%s: page_size must be a power of two >= 64 (got %d), with pages and a table stride", who,
                c->page_size);
      return DFL_ERR_INVALID;
    }
    while ((1 << shift) < c->page_size) ++shift;
  }
  out->k = static_cast<unsigned char*>(c->k);
  out->v = static_cast<unsigned char*>(c->v);
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->seq_stride = c->seq_stride;
  out->head_stride = c->head_stride;
  out->s_seq_stride = c->scale_seq_stride;
  out->s_head_stride = c->scale_head_stride;
  out->page_table = c->page_table;
  out->pt_stride = c->pt_stride;
  out->page_shift = shift;
  out->n_seqs = c->n_seqs;
  out->n_pages = c->n_pages;
  out->cap = c->cap;
  out->Hkv = c->n_kv_heads;
  return DFL_OK;
}

// ---------------------------------------------------------------------------
// Append. hd / 8 lanes per head, eight consecutive values each (one 16-byte load), so a warp holds
// 256 / hd heads (a slot) at a time and a head's sums take log2(hd / 8) shuffles. A CTA takes ROWS
// rows: its threads make the rows' (cos, sin) tables together, then 8 / ROWS warps walk each row's slots, a
// slot's load in flight while the one before it is worked on. Few rows: one row a CTA and its
// slots spread over CTAs (a slot a warp, for latency); many: four rows a CTA.
// ---------------------------------------------------------------------------
struct AppendQ8Args {
  const __nv_bfloat16* qkv;
  long long ldqkv;
  int q_stride;
  const int* pos;
  const int* row_seq;
  const __nv_bfloat16* q_norm;
  const __nv_bfloat16* k_norm;
  const float* inv_freq;
  __nv_bfloat16* q_out;
  Q8Cache c;
  int M, Hq, rot_dim;
  int first_head;  // 0, or Hq when the q heads are left out
  int slots_per_cta;
  float eps;
  int* err;
};

constexpr int APPEND_WARPS = 8;

// cos and sin of p * f: the product and its reduction by turns in fp64 (an fp32 product is off by
// 2^-24 p f, 0.008 rad at position 131072), the reduced angle in fp32.
__device__ __forceinline__ float2 rope_cos_sin(int p, float f) {
  const double a = (double)p * (double)f;
  const double turns = rint(a * 0.15915494309189535);  // 1 / (2 pi)
  float s, c;
  sincosf((float)fma(turns, -6.283185307179586, a), &s, &c);
  return make_float2(c, s);
}

// Codes of four values x * up, rounded to nearest even: int8 by an addition of 1.5 * 2^23, whose sum's low
// byte is the integer (|x * up| <= 127 up to rounding, so none is out of range).
template <bool E4M3>
__device__ __forceinline__ uint32_t q8_codes4(const float* x, float up) {
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * up, x[1] * up), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * up, x[3] * up), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  } else {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[j], up), 12582912.f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
}

template <int HD, bool E4M3, int ROWS>
__global__ void __launch_bounds__(32 * APPEND_WARPS) append_q8_kernel(const __grid_constant__ AppendQ8Args a) {
  grid_dependency_launch_dependents();
  grid_dependency_wait();
  constexpr int LPH = HD / 8;               // lanes per head
  constexpr int HPW = 32 / LPH;             // heads per slot
  constexpr int WPR = APPEND_WARPS / ROWS;  // warps per row
  __shared__ float2 cs[ROWS][HD / 2];
  const int m0 = blockIdx.x * ROWS;
  const int half = a.rot_dim >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = m0 + warp / WPR;
  const int p = m < a.M ? a.pos[m] : -1;
  const int sub = lane / LPH, l = lane % LPH;  // head within the slot, lane within the head
  const int Hkv = a.c.Hkv;
  const int n_heads = a.Hq + 2 * Hkv;
  const __nv_bfloat16* row = a.qkv + (long long)m * a.ldqkv + l * 8;
  const long long kv0 = (long long)a.Hq * a.q_stride;
  auto load = [&](int slot) -> uint4 {
    const int h = slot * HPW + sub;
    if (p < 0 || h < a.first_head || h >= n_heads) return make_uint4(0, 0, 0, 0);
    return *reinterpret_cast<const uint4*>(row + (h < a.Hq ? (long long)h * a.q_stride : kv0 + (long long)(h - a.Hq) * HD));
  };
  const int slots = (n_heads + HPW - 1) / HPW;
  const int slot0 = a.first_head / HPW + blockIdx.y * a.slots_per_cta;
  const int slot_end = min(slots, slot0 + a.slots_per_cta);
  int slot = slot0 + warp % WPR;
  uint4 nx = make_uint4(0, 0, 0, 0);
  if (slot < slot_end) nx = load(slot);
  // tables: thread t makes entries t, t + 256, ... of the CTA's rows
  for (int i = threadIdx.x; i < ROWS * half; i += 32 * APPEND_WARPS) {
    const int r = ROWS == 1 ? 0 : i / half, k = ROWS == 1 ? i : i - r * half;
    const int pr = m0 + r < a.M ? a.pos[m0 + r] : -1;
    if (pr >= 0) cs[r][k] = rope_cos_sin(pr, a.inv_freq[k]);
  }
  __syncthreads();
  if (p < 0 || slot >= slot_end) return;
  const int seq = a.row_seq ? a.row_seq[m] : 0;
  long long page = 0;
  int prow = 0;
  const bool placed = q8_place(a.c, seq, p, lane == 0 ? a.err : nullptr, page, prow);
  // this lane's rotation: its eight values are i .. i + 7 of the first half (partner half / 8
  // lanes up), of the second (down), or behind the rotated dims (turned by 0)
  const int hl = half / 8;
  const bool first = l < hl, second = l >= hl && l < 2 * hl;
  const int src = sub * LPH + (first ? l + hl : second ? l - hl : l);
  float cr[8], sr[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 t = first || second ? cs[warp / WPR][(first ? l : l - hl) * 8 + j] : make_float2(1.f, 0.f);
    cr[j] = t.x;
    sr[j] = first ? -t.y : t.y;  // x' = x cos -/+ partner sin
  }
  const uint4 qw = *reinterpret_cast<const uint4*>(a.q_norm + l * 8);
  const uint4 kw = *reinterpret_cast<const uint4*>(a.k_norm + l * 8);
  const long long code0 = page * a.c.seq_stride + (long long)prow * HD + l * 8;
  const long long scale0 = page * a.c.s_seq_stride + prow;
#pragma unroll 1
  for (; slot < slot_end; slot += WPR) {
    const uint32_t u[4] = {nx.x, nx.y, nx.z, nx.w};
    if (slot + WPR < slot_end) nx = load(slot + WPR);
    const int h = slot * HPW + sub;
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + Hkv;
    const bool live = h >= a.first_head && h < n_heads && (is_q || placed);
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(u[j] << 16);
      x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
    if (slot * HPW < a.Hq + Hkv) {  // some head of the slot is a q or k head: norm and rotation
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = sq_acc(ss, x[j]);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / (float)HD) + a.eps);
      const uint32_t wu[4] = {is_q ? qw.x : kw.x, is_q ? qw.y : kw.y, is_q ? qw.z : kw.z, is_q ? qw.w : kw.w};
      const bool turn = is_q || is_k;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float wj = __uint_as_float(j & 1 ? wu[j >> 1] & 0xffff0000u : wu[j >> 1] << 16);
        const float y = wj * (x[j] * inv);
        const float z = __shfl_sync(0xffffffffu, y, src);
        const float r = __fmaf_rn(y, cr[j], z * sr[j]);
        x[j] = turn ? r : x[j];
      }
    }
    if (is_q && live) {
      uint4 o;
      o.x = pack_bf16x2(x[0], x[1]);
      o.y = pack_bf16x2(x[2], x[3]);
      o.z = pack_bf16x2(x[4], x[5]);
      o.w = pack_bf16x2(x[6], x[7]);
      *reinterpret_cast<uint4*>(a.q_out + ((long long)m * a.Hq + h) * HD + l * 8) = o;
    }
    if (slot * HPW + HPW > a.Hq) {  // some head of the slot is a k or v head: quantise
      // the maximum magnitude as an unsigned comparison of the bits, in which a NaN or an
      // infinity is larger than every finite value
      unsigned am = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) am = max(am, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
      if (!is_q && live) {
        constexpr float TOP = E4M3 ? 448.f : 127.f;
        const bool finite = am < 0x7f800000u;
        const float amax = __uint_as_float(am);
        // below 2^-119 the reciprocal would overflow: such a row is all but zero, and is held as zeros
        const bool some = finite && amax >= 1.5046328e-36f;
        const float up = some ? __fdiv_rn(TOP, amax) : 0.f;
        const float scale = finite ? (some ? __fdiv_rn(amax, TOP) : 0.f) : __uint_as_float(0x7fc00000u);
        const uint32_t c0 = some ? q8_codes4<E4M3>(x, up) : 0u, c1 = some ? q8_codes4<E4M3>(x + 4, up) : 0u;
        const int kh = h - a.Hq - (is_k ? 0 : Hkv);
        *reinterpret_cast<uint2*>((is_k ? a.c.k : a.c.v) + code0 + kh * a.c.head_stride) = make_uint2(c0, c1);
        if (l == 0) (is_k ? a.c.ks : a.c.vs)[scale0 + kh * a.c.s_head_stride] = scale;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read-back: one thread per 16 codes of a key row and of the value row of the same place.
// ---------------------------------------------------------------------------
struct ReadQ8Args {
  Q8Cache c;
  const int* pos;
  const int* row_seq;
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
  long long n;  // threads with work: M * Hkv * hd / 16
  int* err;
};

template <bool E4M3>
__device__ __forceinline__ void q8_values4(uint32_t w, float (&f)[4]) {
  if (E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
      const float2 v = __half22float2(__half2(h));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(signed char)(w >> (8 * i));
  }
}

template <int HD, bool E4M3>
__global__ void __launch_bounds__(256) read_q8_kernel(const __grid_constant__ ReadQ8Args a) {
  grid_dependency_launch_dependents();
  grid_dependency_wait();
  constexpr int CPR = HD / 16;  // 16-code chunks per row
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.n) return;
  const int c = (int)(i % CPR);
  const long long mh = i / CPR;
  const int h = (int)(mh % a.c.Hkv);
  const int m = (int)(mh / a.c.Hkv);
  const int p = a.pos[m];
  if (p < 0) return;
  long long page;
  int row;
  if (!q8_place(a.c, a.row_seq ? a.row_seq[m] : 0, p, c == 0 && h == 0 ? a.err : nullptr, page, row)) return;
  const long long off = page * a.c.seq_stride + h * a.c.head_stride + (long long)row * HD + c * 16;
  const long long soff = page * a.c.s_seq_stride + h * a.c.s_head_stride + row;
  const uint4 kw = __ldg(reinterpret_cast<const uint4*>(a.c.k + off));
  const uint4 vw = __ldg(reinterpret_cast<const uint4*>(a.c.v + off));
  const float ks = __ldg(a.c.ks + soff), vs = __ldg(a.c.vs + soff);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint4 w = t ? vw : kw;
    const float s = t ? vs : ks;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[4];
      q8_values4<E4M3>(u[q], f);
      o[2 * q] = pack_bf16x2(f[0] * s, f[1] * s);
      o[2 * q + 1] = pack_bf16x2(f[2] * s, f[3] * s);
    }
    uint4* dst = reinterpret_cast<uint4*>((t ? a.v_out : a.k_out) + mh * HD + c * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <typename A>
static int launch_q8(void (*kernel)(A), const A& a, dim3 grid, int threads, const char* who, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

}  // namespace dfl

using namespace dfl;

static bool misaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

extern "C" int dfl_qkv_rope_append_q8(const void* qkv, int64_t ldqkv, int q_stride, const int32_t* pos,
                                      const int32_t* row_seq, const void* q_norm, const void* k_norm,
                                      const float* inv_freq, void* q_out, const dfl_kv_q8* cache, int M, int Hq,
                                      int rot_dim, float eps, int do_q, void* stream) {
  const char* who = "dfl_qkv_rope_append_q8";
  if (M == 0) return DFL_OK;
  AppendQ8Args a;
  if (const int s = q8_cache(cache, who, &a.c)) return s;
  const int hd = cache->head_dim;
  if (!qkv || !pos || !k_norm || (rot_dim > 0 && !inv_freq) || (do_q && (!q_out || !q_norm)) || M < 0 || Hq < 0) {
    set_error("%s: null pointer or negative size", who);
    return DFL_ERR_INVALID;
  }
  if (rot_dim < 0 || rot_dim > hd || rot_dim % 16) {
    set_error("%s: rot_dim %d must be a multiple of 16, at most head_dim", who, rot_dim);
    return DFL_ERR_UNSUPPORTED;
  }
  if (misaligned16(qkv) || misaligned16(k_norm) || (do_q && (misaligned16(q_norm) || misaligned16(q_out))) ||
      ldqkv % 8 || q_stride % 8 || q_stride < (Hq ? hd : 0) ||
      ldqkv < (int64_t)Hq * q_stride + 2 * (int64_t)cache->n_kv_heads * hd) {
    set_error("%s: rows, norm weights and q_out must be 16-byte aligned and ldqkv cover a row (ldqkv=%lld)", who,
              (long long)ldqkv);
    return DFL_ERR_UNSUPPORTED;
  }
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.ldqkv = ldqkv;
  a.q_stride = q_stride;
  a.pos = pos;
  a.row_seq = row_seq;
  a.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  a.q_norm = do_q ? static_cast<const __nv_bfloat16*>(q_norm) : a.k_norm;
  a.inv_freq = inv_freq;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.M = M;
  a.Hq = Hq;
  a.rot_dim = rot_dim;
  a.first_head = do_q ? 0 : Hq;
  a.eps = eps;
  a.err = device_error_word();
  const int per_slot = 256 / hd;
  const int slots = (Hq + 2 * cache->n_kv_heads + per_slot - 1) / per_slot;
  // Up to about four CTAs an SM: one row each, its slots over CTAs of eight. Beyond: four rows a CTA
  // (16384 rows of 48 heads of 128: APPEND_TIMES).
  const int groups = (slots - a.first_head / per_slot + APPEND_WARPS - 1) / APPEND_WARPS;
  const bool few = (long long)M * groups <= 148 * 4;
  a.slots_per_cta = few ? APPEND_WARPS : slots;
  const dim3 grid(few ? M : (M + 3) / 4, few ? groups : 1);
  cudaStream_t st = as_stream(stream);
  const int thr = 32 * APPEND_WARPS;
  const bool e4 = cache->type == DFL_KV_E4M3;
#define APPEND_Q8(HD)                                                                                              \
  return few ? launch_q8(e4 ? append_q8_kernel<HD, true, 1> : append_q8_kernel<HD, false, 1>, a, grid, thr, who, st) \
             : launch_q8(e4 ? append_q8_kernel<HD, true, 4> : append_q8_kernel<HD, false, 4>, a, grid, thr, who, st)
  switch (hd) {
    case 64: APPEND_Q8(64);
    case 128: APPEND_Q8(128);
    default: APPEND_Q8(256);
  }
#undef APPEND_Q8
}

extern "C" int dfl_kv_read_q8(const dfl_kv_q8* cache, const int32_t* pos, const int32_t* row_seq, int M, void* k_out,
                              void* v_out, void* stream) {
  const char* who = "dfl_kv_read_q8";
  if (M == 0) return DFL_OK;
  ReadQ8Args a;
  if (const int s = q8_cache(cache, who, &a.c)) return s;
  if (!pos || !k_out || !v_out || M < 0) {
    set_error("%s: null pointer or negative size", who);
    return DFL_ERR_INVALID;
  }
  if (misaligned16(k_out) || misaligned16(v_out)) {
    set_error("%s: outputs must be 16-byte aligned", who);
    return DFL_ERR_UNSUPPORTED;
  }
  const int hd = cache->head_dim;
  a.pos = pos;
  a.row_seq = row_seq;
  a.k_out = static_cast<__nv_bfloat16*>(k_out);
  a.v_out = static_cast<__nv_bfloat16*>(v_out);
  a.n = (long long)M * cache->n_kv_heads * (hd / 16);
  a.err = device_error_word();
  const long long blocks = (a.n + 255) / 256;
  if (blocks > 0x7fffffffLL) {
    set_error("%s: too many rows (%d)", who, M);
    return DFL_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)blocks);
  cudaStream_t st = as_stream(stream);
  const bool e4 = cache->type == DFL_KV_E4M3;
  switch (hd) {
    case 64: return launch_q8(e4 ? read_q8_kernel<64, true> : read_q8_kernel<64, false>, a, grid, 256, who, st);
    case 128: return launch_q8(e4 ? read_q8_kernel<128, true> : read_q8_kernel<128, false>, a, grid, 256, who, st);
    default: return launch_q8(e4 ? read_q8_kernel<256, true> : read_q8_kernel<256, false>, a, grid, 256, who, st);
  }
}
