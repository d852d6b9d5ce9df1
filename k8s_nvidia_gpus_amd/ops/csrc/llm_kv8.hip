// Paged KV cache in 8 bits and the attention that reads it (LLM serving), gfx950.
//
// A page holds 64 positions of every KV head; each (page, head) has one key scale and one value scale:
//   k  [pages][Hkv][64][D]   key codes, position-major         K[j] = ks code
//   v  [pages][Hkv][D][64]   value codes, dim-major            V[j] = vs code
//   ks, vs [pages][Hkv]      fp32, powers of two: the least 2^e with amax <= qmax 2^e (int8 127,
//                            e4m3 448); 0 for an all-zero block, NaN for one with a non-finite value
// Values lie dim-major because the P.V matrix instruction takes, for one dim, consecutive positions of
// a lane: both products then read the cache in the order their operands need it, straight from memory
// (decode) or with plain LDS reads (prompt), and nothing is transposed on the way.
// Scales are powers of two so that code x scale is exact in bf16 and a scale that has to grow (a larger
// value arrives in a begun page) shifts the old codes: an e4m3 page loses only subnormals by it, an
// int8 page at most 1/2 + 1/4 + ... < 1 step however often it grows (with scales of amax / 127 every
// growth would round anew).  The price is a step up to twice as large as amax / 127.
//
// A sequence is a row of the page table; an entry outside the pool (-1) is an unmapped page: what
// would be written there is dropped, and its positions are not attended.  Query p sees key j when
//   j <= p  and  (window == 0 or j > p - window or j < sinks).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace {

constexpr int kPage = 64;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

enum { kF16 = 0, kBF16 = 1, kF32 = 2 };

// ---------------------------------------------------------------- 16-bit and 8-bit types
template <int T>
struct Elem;
template <>
struct Elem<kF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
template <>
struct Elem<kBF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
template <>
struct Elem<kF32> {
  typedef float type;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

// 16 bytes that nobody reads again soon: non-temporal, so that they leave the caches to others.  Only where
// an instruction takes whole 128-byte lines; the rest of a line in pieces is fetched again.
typedef unsigned u4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load16_once(const void* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(static_cast<const u4v*>(p)));
}

// N consecutive elements as floats; `wide`: the address is a multiple of 16 bytes (uniform)
template <int T, int N>
__device__ __forceinline__ void load_n(const typename Elem<T>::type* p, bool wide, float (&x)[N]) {
  typedef typename Elem<T>::type E;
  constexpr int PER = 16 / sizeof(E);
  if (wide) {
#pragma unroll
    for (int c = 0; c < N / PER; ++c) {
      const uint4 w = reinterpret_cast<const uint4*>(p)[c];
      E e[PER];
      __builtin_memcpy(e, &w, 16);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[c * PER + i] = Elem<T>::get(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = Elem<T>::get(p[i]);
  }
}
// ONCE: non-temporal
template <int T, int N, bool ONCE = false>
__device__ __forceinline__ void store_n(typename Elem<T>::type* p, bool wide, const float (&x)[N]) {
  typedef typename Elem<T>::type E;
  constexpr int PER = 16 / sizeof(E);
  if (wide) {
#pragma unroll
    for (int c = 0; c < N / PER; ++c) {
      E e[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) e[i] = Elem<T>::put(x[c * PER + i]);
      u4v w;
      __builtin_memcpy(&w, e, 16);
      if constexpr (ONCE) __builtin_nontemporal_store(w, reinterpret_cast<u4v*>(p) + c);
      else reinterpret_cast<u4v*>(p)[c] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = Elem<T>::put(x[i]);
  }
}

// four codes of one dword as fp16 pairs (exact: |int8| < 2^11, e4m3 has 4 significant bits and fp16's
// exponent range).  int8: the byte with its sign flipped is code + 128; under the high byte 0x64 it
// reads as the fp16 1024 + 128 + code, and one packed subtraction leaves the code.
template <bool FP8>
__device__ __forceinline__ void codes_h4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, a) - bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, b) - bias);
  }
}
// eight codes (two dwords) as the eight fp16 of a matrix operand
template <bool FP8>
__device__ __forceinline__ h8 codes_h8(uint32_t a, uint32_t b) {
  uint4 r;
  codes_h4<FP8>(a, r.x, r.y);
  codes_h4<FP8>(b, r.z, r.w);
  return __builtin_bit_cast(h8, r);
}
template <bool FP8>
__device__ __forceinline__ void codes_f4(uint32_t w, float (&x)[4]) {
  if constexpr (FP8) {
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
}
// four values (already divided by the scale) to codes, ties to even
template <bool FP8>
__device__ __forceinline__ uint32_t to_codes4(float a, float b, float c, float d) {
  if constexpr (FP8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    return ((uint32_t)(int)__builtin_rintf(a) & 0xffu) | (((uint32_t)(int)__builtin_rintf(b) & 0xffu) << 8) |
           (((uint32_t)(int)__builtin_rintf(c) & 0xffu) << 16) | ((uint32_t)(int)__builtin_rintf(d) << 24);
  }
}
template <bool FP8>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  float x[4];
  codes_f4<FP8>(w, x);
  return to_codes4<FP8>(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
}

// four dwords as a 4 x 4 matrix of bytes, transposed
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// the least 2^e with amax <= qmax 2^e, from amax's bits (>= 0; NaN and infinity have the largest)
template <bool FP8>
__device__ __forceinline__ float block_scale(uint32_t bits) {
  if (bits == 0) return 0.f;
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int ex = (int)(bits >> 23) - 127;              // a subnormal amax falls under the floor below
  // qmax = 1.984375 x 2^6 (127) or 1.75 x 2^8 (448): one more when the significand passes it
  const int e = FP8 ? ex - 8 + ((bits & 0x7fffffu) > 0x600000u) : ex - 6 + ((bits & 0x7fffffu) > 0x7e0000u);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// ---------------------------------------------------------------- across a wave
// Inclusive scan of 64 lanes in six data-parallel-primitive steps (rows of 16, then across rows): a few
// cycles each, where a shuffle takes an LDS round trip.  The last lane has the whole wave's.
template <typename F>
__device__ __forceinline__ int wave_scan(int x, int none, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x111, 0xf, 0xf, false));   // row_shr:1
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x112, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x114, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x118, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x142, 0xa, 0xf, false));   // row_bcast:15
  x = f(x, __builtin_amdgcn_update_dpp(none, x, 0x143, 0xc, 0xf, false));   // row_bcast:31
  return x;
}

__device__ __forceinline__ float wave_max(float x) {
  const int r = wave_scan(__float_as_int(x), (int)0xff800000, [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  });
  return __int_as_float(__builtin_amdgcn_readlane(r, 63));
}
__device__ __forceinline__ float wave_sum(float x) {
  const int r = wave_scan(__float_as_int(x), 0, [](int a, int b) {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  });
  return __int_as_float(__builtin_amdgcn_readlane(r, 63));
}

// ---------------------------------------------------------------- ragged segments
// Sequence s has rows cu[s] .. cu[s + 1] - 1 at positions start[s] ..; what is out of order, out of
// [0, N) or at a negative start counts as empty.
struct Segs {
  const int* start;
  const int* cu;
  int S, N;
  __device__ __forceinline__ void get(int s, int& row, int& n, int& pos) const {
    row = max(cu[s], 0);
    n = max(min(cu[s + 1], N), 0) - row;
    pos = start[s];
    if (pos < 0 || pos > 0x3fffffff) n = 0;
  }
};

// A piece of a segment: the segment, its rows (row .. row + cnt - 1, at pos ..) and the piece's index.
struct Piece {
  int s, index, row, cnt, pos;
};
// The unit'th piece of all segments, each cut into pieces by `count` (pieces of n rows at pos); the whole
// wave calls it and gets the same answer.  False: there are fewer pieces.
template <typename F>
__device__ __forceinline__ bool find_piece(const Segs& sg, int unit, F count, Piece& out) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < sg.S; base += 64) {
    int c = 0, row = 0, n = 0, pos = 0;
    if (base + lane < sg.S) {
      sg.get(base + lane, row, n, pos);
      c = n > 0 ? count(n, pos) : 0;
    }
    const int inc = wave_scan(c, 0, [](int a, int b) { return a + b; });
    const uint64_t past = __ballot(before + inc > unit);
    if (past) {
      const int hit = __builtin_ctzll(past);
      out.s = base + hit;
      out.index = unit - before - (__builtin_amdgcn_readlane(inc, hit) - __builtin_amdgcn_readlane(c, hit));
      out.row = __builtin_amdgcn_readlane(row, hit);
      out.cnt = __builtin_amdgcn_readlane(n, hit);
      out.pos = __builtin_amdgcn_readlane(pos, hit);
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, 63);
  }
  return false;
}

// The segment that row n is in (the whole wave asks for one row): its rows row .. end - 1, at pos ...  False,
// and end = 0: none.
struct Row {
  int row, end, pos;
};
__device__ __forceinline__ bool find_row(const Segs& sg, int n, Row& out) {
  const int lane = threadIdx.x & 63;
  int s = 0;                                             // segments that end at or before row n
  for (int base = 0; base < sg.S; base += 64)
    s += __builtin_popcountll(__ballot(base + lane < sg.S && sg.cu[base + lane + 1] <= n));
  s = __builtin_amdgcn_readfirstlane(s);
  out = Row{0, 0, 0};
  if (s >= sg.S) return false;
  int cnt;
  sg.get(s, out.row, cnt, out.pos);
  const bool in = n >= out.row && n < out.row + cnt;
  out.end = in ? out.row + cnt : 0;
  return in;
}

__device__ __forceinline__ int pages_of(int n, int pos) { return (pos + n - 1) / kPage - pos / kPage + 1; }

// most pages that N rows in S segments touch, whatever their positions
inline long most_pages(long N, long S) {
  const long m = (N + 62 * S) / 64 + S;
  return m < N ? m : N;
}

struct Pool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  const int* table;
  int pool, Hkv, width, stride;        // pages in the pool; table columns and row stride
  __device__ __forceinline__ int page(int s, int j) const {
    if ((unsigned)j >= (unsigned)width) return -1;
    const int id = table[(long)s * stride + j];
    return (unsigned)id < (unsigned)pool ? id : -1;
  }
};

// ---------------------------------------------------------------- append
struct AppendArgs {
  Pool c;
  Segs sg;
  const void* k;
  const void* v;
  const void* q;
  void* qo;
  const float* cos_t;
  const float* sin_t;
  long sk_tok, sk_head, sv_tok, sv_head, sq_tok, sq_head, so_tok, so_head;
  int H, units, per, table_rows;       // per: query rows a wave; table_rows: rows of the rotation tables
  bool wide_kv, wide_q;
};

// a rounding after every operation (the compiler would fuse the products into one fma otherwise)
__device__ __forceinline__ float turn_lo(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * c, y = b * s;
  return x - y;
}
__device__ __forceinline__ float turn_hi(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * s, y = b * c;
  return x + y;
}

// eight pairs (d, d + D/2) of one row, and their rotation
template <int T, int D>
__device__ __forceinline__ void load_pairs(const typename Elem<T>::type* row, bool wide, int d0, float (&lo)[8],
                                           float (&hi)[8]) {
  load_n<T, 8>(row + d0, wide, lo);
  load_n<T, 8>(row + D / 2 + d0, wide, hi);
}
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = lo[i], b = hi[i];
    lo[i] = turn_lo(a, b, c[i], s[i]);
    hi[i] = turn_hi(a, b, c[i], s[i]);
  }
}

// Blocks [0, units * Hkv): one page of one sequence and KV head each, 256 threads: the new rows' keys
// are rotated, the page's new scale is the larger of the old one (if the page was begun before) and
// the new rows' own, old codes are shifted if it grew, the new rows' codes are written.  One block owns
// the page's codes and scales, so there are no atomics.  The blocks behind rotate the queries, `per` rows
// a wave, a lane's pairs the same in every head (its table entries are read once a row).  Memory-bound:
// 16-byte loads and stores of whole rows; values change their order on the way, through LDS and 4 x 4
// byte transposes in registers, eight lanes writing a dim's 64 positions.  12800 tokens of 28 + 4 + 4
// heads behind 8 x 1500: 55 us, 4.0 TB/s (14 us without the queries); a token for each of 4 sequences
// 5.5 us, of it about 2 us the launch: segment search, page entry and scale, the block's maximum and the
// stores wait for each other.
template <int D, bool FP8, int T, int TO>
__global__ void __launch_bounds__(256) kv8_append_kernel(const AppendArgs a) {
  typedef typename Elem<T>::type E;
  constexpr int PR = D / 16;                             // 8-pair items of a row
  constexpr int PER = kPage * PR / 256;                  // items a thread
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x >= a.units * a.c.Hkv) {            // ---- queries: a.per rows a wave
    typedef typename Elem<TO>::type EO;
    const int d0 = 8 * (lane % PR);                        // a lane's pairs, of every 64 / PR'th head
    const int n0 = (((int)blockIdx.x - a.units * a.c.Hkv) * 4 + wave) * a.per;
    Row at{0, 0, 0};
    for (int n = n0; n < min(n0 + a.per, a.sg.N); ++n) {
      if (n >= at.end && !find_row(a.sg, n, at)) continue;
      const int pos = at.pos + n - at.row;
      if (pos >= a.table_rows) continue;
      const E* q = static_cast<const E*>(a.q) + (long)n * a.sq_tok;
      EO* o = static_cast<EO*>(a.qo) + (long)n * a.so_tok;
      float c[8], s[8];
      if (a.cos_t) {
        load_n<kF32, 8>(a.cos_t + (long)pos * (D / 2) + d0, true, c);
        load_n<kF32, 8>(a.sin_t + (long)pos * (D / 2) + d0, true, s);
      }
#pragma unroll 4
      for (int h = lane / PR; h < a.H; h += 64 / PR) {
        float lo[8], hi[8];
        load_pairs<T, D>(q + h * a.sq_head, a.wide_q, d0, lo, hi);
        if (a.cos_t) turn(lo, hi, c, s);
        store_n<TO, 8>(o + h * a.so_head + d0, a.wide_q, lo);
        store_n<TO, 8>(o + h * a.so_head + D / 2 + d0, a.wide_q, hi);
      }
    }
    return;
  }
  __shared__ uint32_t red[2][4];
  __shared__ __align__(8) uint8_t img[kPage][D + 8];     // value codes by position
  const int kh = blockIdx.x % a.c.Hkv;
  Piece pc;
  if (!find_piece(a.sg, blockIdx.x / a.c.Hkv, [](int n, int p) { return pages_of(n, p); }, pc)) return;
  const int pos = pc.pos, cnt = pc.cnt, row = pc.row;
  const int j = pos / kPage + pc.index;
  if (j >= a.c.width) return;                            // behind the table (and its rotation tables)
  const int r0 = max(pos - j * kPage, 0), r1 = min(pos + cnt - j * kPage, kPage);   // new rows
  const long n0 = (long)row + j * kPage - pos;           // input row of the page's position 0
  const E* kin = static_cast<const E*>(a.k) + kh * a.sk_head;
  const E* vin = static_cast<const E*>(a.v) + kh * a.sv_head;
  // the inputs do not wait for the table entry
  float klo[PER][8] = {}, khi[PER][8] = {}, vlo[PER][8] = {}, vhi[PER][8] = {}, cs[PER][8] = {}, sn[PER][8] = {};
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = tid + 256 * u, r = i / PR, d0 = 8 * (i % PR);
    if (r < r0 || r >= r1) continue;
    load_pairs<T, D>(kin + (n0 + r) * a.sk_tok, a.wide_kv, d0, klo[u], khi[u]);
    load_n<T, 8>(vin + (n0 + r) * a.sv_tok + 2 * d0, a.wide_kv, vlo[u]);
    load_n<T, 8>(vin + (n0 + r) * a.sv_tok + 2 * d0 + 8, a.wide_kv, vhi[u]);
    if (a.cos_t) {
      load_n<kF32, 8>(a.cos_t + ((long)j * kPage + r) * (D / 2) + d0, true, cs[u]);
      load_n<kF32, 8>(a.sin_t + ((long)j * kPage + r) * (D / 2) + d0, true, sn[u]);
    }
  }
  const int id = a.c.page(pc.s, j);
  if (id < 0) return;
  const long sc = (long)id * a.c.Hkv + kh;
  uint8_t* kc = a.c.k + sc * kPage * D;
  uint8_t* vc = a.c.v + sc * kPage * D;
  const float oldk = r0 ? a.c.ks[sc] : 0.f, oldv = r0 ? a.c.vs[sc] : 0.f;
  // old value codes of 8 positions of 4 dims, where some of those are not new
  constexpr int PV = D * 2 / 256 + (D * 2 % 256 != 0);
  uint2 was[PV][4] = {};
#pragma unroll
  for (int u = 0; u < PV; ++u) {
    const int i = tid + 256 * u, p0 = 8 * (i & 7), d = 4 * (i >> 3);
    if (d < D && p0 < r1 && (p0 < r0 || p0 + 8 > r1)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) was[u][e] = *reinterpret_cast<const uint2*>(vc + (d + e) * kPage + p0);
    }
  }
  uint32_t mk = 0, mv = 0;                               // largest magnitudes, as bits (NaN largest)
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (a.cos_t) turn(klo[u], khi[u], cs[u], sn[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mk = max(mk, max(__float_as_uint(klo[u][e]) & 0x7fffffffu, __float_as_uint(khi[u][e]) & 0x7fffffffu));
      mv = max(mv, max(__float_as_uint(vlo[u][e]) & 0x7fffffffu, __float_as_uint(vhi[u][e]) & 0x7fffffffu));
    }
  }
  mk = wave_scan(mk, 0, [](int a, int b) { return max(a, b); });   // (31 bits: they order as integers do)
  mv = wave_scan(mv, 0, [](int a, int b) { return max(a, b); });
  if (lane == 63) { red[0][wave] = mk; red[1][wave] = mv; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) { mk = max(mk, red[0][w]); mv = max(mv, red[1][w]); }
  // the larger of both, NaN above all (scales are never negative: their bits order like they do)
  const float nk = __uint_as_float(max(__float_as_uint(block_scale<FP8>(mk)), __float_as_uint(oldk)));
  const float nv = __uint_as_float(max(__float_as_uint(block_scale<FP8>(mv)), __float_as_uint(oldv)));
  const float ik = nk > 0.f ? 1.f / nk : 0.f, iv = nv > 0.f ? 1.f / nv : 0.f;
  const bool badk = nk != nk, badv = nv != nv;
  const bool growk = r0 && nk > oldk, growv = r0 && nv > oldv;   // (a NaN block keeps its codes)
  if (tid == 0) { a.c.ks[sc] = nk; a.c.vs[sc] = nv; }
  if (growk) {
    const float ratio = oldk * ik;
    for (int i = tid; i < r0 * (D / 16); i += 256) {
      uint4 w = reinterpret_cast<uint4*>(kc)[i];
      w.x = rescale4<FP8>(w.x, ratio); w.y = rescale4<FP8>(w.y, ratio);
      w.z = rescale4<FP8>(w.z, ratio); w.w = rescale4<FP8>(w.w, ratio);
      reinterpret_cast<uint4*>(kc)[i] = w;
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = tid + 256 * u, r = i / PR, d0 = 8 * (i % PR);
    if (r >= r0 && r < r1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        klo[u][e] = badk ? 0.f : klo[u][e] * ik;
        khi[u][e] = badk ? 0.f : khi[u][e] * ik;
        vlo[u][e] = badv ? 0.f : vlo[u][e] * iv;
        vhi[u][e] = badv ? 0.f : vhi[u][e] * iv;
      }
      auto eight = [&](const float (&x)[8]) {
        return make_uint2(to_codes4<FP8>(x[0], x[1], x[2], x[3]), to_codes4<FP8>(x[4], x[5], x[6], x[7]));
      };
      *reinterpret_cast<uint2*>(kc + r * D + d0) = eight(klo[u]);
      *reinterpret_cast<uint2*>(kc + r * D + D / 2 + d0) = eight(khi[u]);
      *reinterpret_cast<uint2*>(&img[r][2 * d0]) = eight(vlo[u]);
      *reinterpret_cast<uint2*>(&img[r][2 * d0 + 8]) = eight(vhi[u]);
    }
  }
  __syncthreads();
  // 8 positions of 4 dims a thread: eight lanes write a dim's 64 bytes
  const float rv = growv ? oldv * iv : 1.f;
#pragma unroll
  for (int u = 0; u < PV; ++u) {
    const int i = tid + 256 * u, p0 = 8 * (i & 7), d = 4 * (i >> 3);
    const bool has_new = p0 < r1 && p0 + 8 > r0;
    if (d >= D || (!has_new && !(growv && p0 < r0))) continue;
    uint32_t lo[4], hi[4];                               // by position, then (transposed) by dim
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = *reinterpret_cast<const uint32_t*>(&img[p0 + e][d]);
      hi[e] = *reinterpret_cast<const uint32_t*>(&img[p0 + 4 + e][d]);
    }
    transpose4(lo);
    transpose4(hi);
    uint32_t keep[2] = {0, 0};                           // bytes that are not new
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (p0 + e < r0 || p0 + e >= r1) keep[e >> 2] |= 0xffu << (8 * (e & 3));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint2* at = reinterpret_cast<uint2*>(vc + (d + e) * kPage + p0);
      uint2 w = make_uint2(lo[e], hi[e]);
      if (keep[0] | keep[1]) {
        uint2 old = was[u][e];
        if (growv) { old.x = rescale4<FP8>(old.x, rv); old.y = rescale4<FP8>(old.y, rv); }
        w.x = (w.x & ~keep[0]) | (old.x & keep[0]);
        w.y = (w.y & ~keep[1]) | (old.y & keep[1]);
      }
      *at = w;
    }
  }
}

// ---------------------------------------------------------------- read
struct ReadArgs {
  Pool c;
  Segs sg;
  void* ko;
  void* vo;
  long sk_tok, sk_head, sv_tok, sv_head;
  bool wide;
};

// One page of one sequence and KV head a block: keys row by row, values through byte transposes and LDS.
// Memory-bound, with 16-bit rows two thirds of the bytes stores: 8 x 16384 positions 56 us, 5.2 TB/s (a copy
// reaches as much); through the caches (key codes in, rows out) 68.
template <int D, bool FP8, int T>
__global__ void __launch_bounds__(256) kv8_read_kernel(const ReadArgs a) {
  typedef typename Elem<T>::type E;
  __shared__ __align__(8) uint8_t img[kPage][D + 8];     // value codes by position
  constexpr int PK = kPage * D / 16 / 256, PV = D * 2 / 256 + (D * 2 % 256 != 0);
  const int tid = threadIdx.x;
  const int kh = blockIdx.x % a.c.Hkv;
  Piece pc;
  if (!find_piece(a.sg, blockIdx.x / a.c.Hkv, [](int n, int p) { return pages_of(n, p); }, pc)) return;
  const int pos = pc.pos, cnt = pc.cnt, row = pc.row;
  const int j = pos / kPage + pc.index;
  const int r0 = max(pos - j * kPage, 0), r1 = min(pos + cnt - j * kPage, kPage);
  const long n0 = (long)row + j * kPage - pos;
  const int id = a.c.page(pc.s, j);
  const bool live = id >= 0;
  const long sc = (long)max(id, 0) * a.c.Hkv + kh;       // an unmapped page: page 0, times 0 (and no NaN code)
  const uint8_t* kc = a.c.k + sc * kPage * D;
  const uint8_t* vc = a.c.v + sc * kPage * D;
  const float sk = live ? a.c.ks[sc] : 0.f, sv = live ? a.c.vs[sc] : 0.f;
  const uint32_t mask = live ? ~0u : 0u;
  uint4 kx[PK];
#pragma unroll
  for (int u = 0; u < PK; ++u) kx[u] = load16_once(kc + 16 * (tid + 256 * u));
  uint2 vx[PV][4];                                       // 8 positions of 4 dims
#pragma unroll
  for (int u = 0; u < PV; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = tid + 256 * u, d = 4 * (i >> 3);
      if (d < D) vx[u][e] = *reinterpret_cast<const uint2*>(vc + (d + e) * kPage + 8 * (i & 7));
    }
  auto put = [&](E* out, const uint32_t (&w)[4], float scale) __attribute__((always_inline)) {
    float y[16], x[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      codes_f4<FP8>(w[c] & mask, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[4 * c + e] = x[e] * scale;
    }
    store_n<T, 16, true>(out, a.wide, y);
  };
#pragma unroll
  for (int u = 0; u < PK; ++u) {
    const int i = tid + 256 * u, r = i / (D / 16), d0 = 16 * (i % (D / 16));
    const uint32_t w[4] = {kx[u].x, kx[u].y, kx[u].z, kx[u].w};
    if (r >= r0 && r < r1) put(static_cast<E*>(a.ko) + (n0 + r) * a.sk_tok + kh * a.sk_head + d0, w, sk);
  }
#pragma unroll
  for (int u = 0; u < PV; ++u) {
    const int i = tid + 256 * u, p0 = 8 * (i & 7), d = 4 * (i >> 3);
    if (d >= D) continue;
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { lo[e] = vx[u][e].x; hi[e] = vx[u][e].y; }
    transpose4(lo);
    transpose4(hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      *reinterpret_cast<uint32_t*>(&img[p0 + e][d]) = lo[e];
      *reinterpret_cast<uint32_t*>(&img[p0 + 4 + e][d]) = hi[e];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PK; ++u) {
    const int i = tid + 256 * u, r = i / (D / 16), d0 = 16 * (i % (D / 16));
    if (r < r0 || r >= r1) continue;
    const uint2 a0 = *reinterpret_cast<const uint2*>(&img[r][d0]), a1 = *reinterpret_cast<const uint2*>(&img[r][d0 + 8]);
    const uint32_t w[4] = {a0.x, a0.y, a1.x, a1.y};
    put(static_cast<E*>(a.vo) + (n0 + r) * a.sv_tok + kh * a.sv_head + d0, w, sv);
  }
}

// ---------------------------------------------------------------- attention, both forms
// The pages that queries at positions lo .. hi see, as a list: the first `sinks` ones, then those from
// `first` on.  For one query each of them has a key that it sees (decode counts on it: the page's value scale
// and poison are the row's).
struct Seen {
  int nsink, first, n;
  __device__ __forceinline__ int page(int i) const { return i < nsink ? i : first + i - nsink; }
};
__host__ __device__ __forceinline__ Seen seen_pages(int lo, int hi, int span, int window, int sinks) {
  Seen s{0, 0, 0};
  const int end = hi < span ? hi + 1 : span;             // keys below `end`
  if (end <= 0) return s;
  const int last = (end + kPage - 1) / kPage;
  if (window > 0) {
    const int low = lo - window + 1;
    s.first = low > 0 ? low / kPage : 0;
    if (low >= end) s.first = last;                      // (no key of page low / kPage lies in the window)
    const int ns = sinks < end ? (sinks + kPage - 1) / kPage : last;
    s.nsink = ns < s.first ? ns : s.first;
  }
  s.n = s.nsink + last - s.first;
  return s;
}

// x of lane l ^ 16 / l ^ 32 on the VALU
__device__ __forceinline__ float xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Factor of a page's raw scores (codes x fitted query) to log2 units, ks the page's key scale and c the
// query's own (>= 0).  Never 0: a masked score is -inf, and 0 x -inf would be NaN; the raw scores of a
// zero page are 0, whatever the factor.  NaN stays.
__device__ __forceinline__ float score_factor(float ks, float c) {
  const float f = ks * c;
  return f < 1e-37f ? 1e-37f : f;
}
// log2 of a page's value scale over the reference `vref` (the largest that the row has seen, > 0 unless all
// were 0).
// The weights p = 2^(s - m) go to the matrix instruction as fp16 p vs / vref, so that pages of unlike
// scales add up in one accumulator; the sum of the plain p's takes the factor back (`back`).  A zero
// page has zero codes: any weight will do.  A NaN scale stays.  What the rounding costs: 2^-11 of a weight,
// and what is below 2^-32 of the largest weight times the largest value scale is lost.  For the reference
// maximum lies up to 8 below the true one (rescaling is put off that long) and the exponents have kBias
// added: the largest weight is 2^7 to 2^15, under fp16's largest, and half of fp16's least step is 2^-25.
constexpr float kDefer = 8.f, kBias = 7.f;
__device__ __forceinline__ float value_weight(float vs, float ratio, float& back) {   // ratio: vs / vref
  float lw = vs == 0.f ? 0.f : __builtin_amdgcn_logf(ratio);
  lw = lw < -60.f ? -60.f : lw;                          // no fp16 weight is left there anyway
  back = __builtin_amdgcn_exp2f(-lw);
  return lw;
}

// a power of two f so that x f (|x| <= amax) has fp16's range to spare: amax f in [2^8, 2^9)
__device__ __forceinline__ float fit_f16(float amax) {
  const int ex = (int)((__float_as_uint(amax) >> 23) & 0xff);
  return ex == 0 || ex == 255 ? 1.f : __uint_as_float((uint32_t)(min(max(262 - ex, 1), 254)) << 23);
}

struct AttnArgs {
  Pool c;
  Segs sg;                 // prompt; decode: start = positions, N = S
  const uint16_t* q;
  void* out;               // null: only q8
  float* po;               // partial outputs [parts][rows][H][D], rows = N
  float* pml;              // [parts][rows][H][2] (max in log2 units, sum)
  int8_t* x8;              // Q8 output (decode): [N][H D], scales of 32, scaled sums of 16
  float* dx;
  float* sx;
  long sq_tok, sq_head, so_tok, so_head;
  int H, G, D, span, window, sinks, parts, units;
  int per;                 // decode: pages a wave (at most 64)
  float c2, sign;          // |scale| x log2(e), and its sign (goes into the query)
  bool wide_q, wide_o;
};

// N consecutive output values at column `col` of row t as Q8: int8 with a scale for each 32 columns and
// the scaled sum of each 16 (neighbouring lanes hold neighbouring columns; blocks begin at lane groups).
template <int N>
__device__ __forceinline__ void put_q8(const AttnArgs& a, int t, long col, const float (&y)[N]) {
  const long at = (long)t * a.H * a.D + col;
  uint32_t top = 0;                                      // as bits: a NaN makes its block's scale NaN
#pragma unroll
  for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 16 / N; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  const float d = __uint_as_float(top) / 127.f;
  int sum = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int c = d > 0.f ? (int)__builtin_rintf(y[e] / d) : 0;
    a.x8[at + e] = (int8_t)c;
    sum += c;
  }
#pragma unroll
  for (int o = 8 / N; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((col & 31) == 0) a.dx[at >> 5] = d;
  if ((col & 15) == 0) a.sx[at >> 4] = d * (float)sum;
}

// Single-token attention.  Grid (Hkv x groups of 16 heads, parts, S); workgroup part p streams pages
// p NW per .. of the row's list, each wave whole pages with its own online softmax, no LDS and no barrier
// until the waves merge.  Both products on v_mfma_f32_16x16x32_f16, operands straight from memory:
// * S = K q^T: tile t of four has the rows m = 0..15 at positions 16 (m >> 2) + 4 t + (m & 3), so that
//   lane (head pr, group kg) gets the scores of positions 16 kg .. 16 kg + 15 over the four tiles;
// * O^T = V^T P^T: the value codes lie dim-major, a lane's 16 bytes are positions 16 kg .. + 15 of one
//   dim: the same positions as its scores, so neither P nor V moves between lanes.  The running
//   maximum, sum and rescaling are one head's, a lane's own.
// A page's keys are loaded as soon as the last page's have been used, and its values likewise: 16 KB in
// flight a wave most of the time at half the registers of two buffers, so three waves fit a SIMD (two
// buffers left one; 32 x 16000 with a window 140 us, this 61, with what follows 51).  ONCE: up to 16 heads
// a KV head, so that no other workgroup of the row reads the page; its values are loaded past the caches
// (8 x 32768 44 -> 40 us, with the window 61 -> 57; with 128 heads on one KV head 14.5 -> 16.6).  Pages that
// sequences share are then fetched past them by each, which costs nothing: with three quarters of every row
// shared 8 x 32000 35.1 us, through the caches 36.0; 32 x 4000 22.3 and 22.0.  Bound by the cache's bytes:
// 8 x 32768 in e4m3 40 us, 5.3 TB/s, where a kernel that only reads reaches 6.5; short contexts by launches
// (two, 2 to 3 us each) and the chain position, page entry, page, join: 8 x 4096 13.4 us, 500 positions 8.1.
template <int D, bool FP8, int T, int NW, bool ONCE>
__global__ void __launch_bounds__(64 * NW, 3) kv8_decode_kernel(const AttnArgs a) {
  constexpr int KH = D / 64, ND = D / 16;
  const int hg = (a.G + 15) / 16;
  const int kh = blockIdx.x / hg, h0 = (blockIdx.x % hg) * 16;
  const int part = blockIdx.y, t = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pr = lane & 15, kg = lane >> 4;
  const int gn = min(16, a.G - h0);                      // heads of this workgroup
  const int p0 = part * a.per * NW;
  const int pos = a.sg.start[t];
  // lane i: table entry and scales of this wave's i'th page (pages p0 + wave + NW i of the list).
  // Without a window the list is the table itself: its entry does not wait for the position.
  int my_id = -1;
  if (a.window <= 0 && lane < a.per) my_id = a.c.page(t, p0 + wave + NW * lane);
  const Seen seen = seen_pages(pos, pos, a.span, a.window, a.sinks);
  const int mine = max(0, min(a.per, (seen.n - p0 - wave + NW - 1) / NW));
  if (a.window > 0 && lane < mine) my_id = a.c.page(t, seen.page(p0 + wave + NW * lane));
  if (part > 0 && p0 >= seen.n) {                        // nothing of the row here: an empty partial
    if ((int)threadIdx.x < gn) {
      float* ml = a.pml + 2 * (((long)part * a.sg.N + t) * a.H + kh * a.G + h0 + threadIdx.x);
      ml[0] = -INFINITY;
      ml[1] = 0.f;
    }
    return;
  }
  float my_ks = 0.f, my_vs = 0.f;
  if (lane < mine && my_id >= 0) {
    const long sc = (long)my_id * a.c.Hkv + kh;
    my_ks = a.c.ks[sc];
    my_vs = a.c.vs[sc];
  }
  uint4 kr[4 * KH], vr[ND];
  auto load_keys = [&](int i) __attribute__((always_inline)) {
    const long id = max(__builtin_amdgcn_readlane(my_id, i), 0);
    const uint8_t* kp = a.c.k + (id * a.c.Hkv + kh) * (kPage * D) + (16 * (pr >> 2) + (pr & 3)) * D + 16 * kg;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int h = 0; h < KH; ++h) kr[u * KH + h] = *reinterpret_cast<const uint4*>(kp + 4 * u * D + 64 * h);
  };
  auto load_values = [&](int i) __attribute__((always_inline)) {
    const long id = max(__builtin_amdgcn_readlane(my_id, i), 0);
    const uint8_t* vp = a.c.v + (id * a.c.Hkv + kh) * (kPage * D) + pr * kPage + 16 * kg;
#pragma unroll
    for (int n = 0; n < ND; ++n)
      vr[n] = ONCE ? load16_once(vp + 16 * n * kPage) : *reinterpret_cast<const uint4*>(vp + 16 * n * kPage);
  };
  if (mine > 0) {
    load_keys(0);
    load_values(0);
  }

  // q operand: head pr, dims 64 h + 16 kg + 8 u + 0..7 (the order in which the key bytes lie)
  h8 qa[2 * KH];
  float qf = a.c2;
  {
    const uint16_t* qr = a.q + (long)t * a.sq_tok + (long)(kh * a.G + h0 + min(pr, gn - 1)) * a.sq_head;
    float x[KH][16], amax = 0.f;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      load_n<T, 16>(qr + 64 * h + 16 * kg, a.wide_q, x[h]);
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[h][e]));
    }
    float f = 1.f;
    if constexpr (T == kBF16) {                          // bf16 to fp16: exact after a shift by head
      amax = fmaxf(amax, xor16(amax));
      amax = fmaxf(amax, xor32(amax));
      f = fit_f16(amax);
      qf /= f;
    }
    f *= a.sign;
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) qa[2 * h + u][e] = (_Float16)(x[h][8 * u + e] * f);
  }

  float m = -INFINITY, l = 0.f, vref = 0.f;
  f4 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f4{0.f, 0.f, 0.f, 0.f};

  const int last = min(pos, a.span - 1);
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    const bool more = i + 1 < mine;
    const bool mapped = __builtin_amdgcn_readlane(my_id, i) >= 0;
    const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_ks), i));
    const float vs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_vs), i));
    const int base = seen.page(p0 + wave + NW * i) * kPage;
    f4 acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      acc[u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        const uint4 w = kr[u * KH + h];
        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h8<FP8>(w.x, w.y), qa[2 * h], acc[u], 0, 0, 0);
        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h8<FP8>(w.z, w.w), qa[2 * h + 1], acc[u], 0, 0, 0);
      }
    }
    if (more) load_keys(i + 1);
    if (!mapped) {                                       // (uniform)
      if (more) load_values(i + 1);
      continue;
    }
    const float f = score_factor(ks, qf);
    float sc[16];                                        // raw: times f in log2 units
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = acc[e >> 2][e & 3];
    const bool whole = base + kPage - 1 <= last &&
                       (a.window <= 0 || base > pos - a.window || base + kPage <= a.sinks);
    if (!whole) {                                        // a border inside the page (wave-uniform)
      const int at = base + 16 * kg, hi = last - at;     // of the registers' own offsets
      const int lo = (a.window > 0 ? pos - a.window : -1) - at, sinks = a.sinks - at;
      uint32_t keep[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool in = (e <= hi) & ((e > lo) | (e < sinks));
        sc[e] = in ? sc[e] : -INFINITY;
        keep[e >> 2] |= in ? 0xffu << (8 * (e & 3)) : 0u;
      }
#pragma unroll
      for (int n = 0; n < ND; ++n) {                     // codes never written may be NaN: 0 x NaN
        vr[n].x &= keep[0]; vr[n].y &= keep[1]; vr[n].z &= keep[2]; vr[n].w &= keep[3];
      }
    }
    float mx = sc[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[e]);
    mx *= f;
    if (vs > vref) {                                     // uniform
      if (vref > 0.f) {
        const float r = vref / vs;
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] *= r;
      }
      vref = vs;
    }
    // rescale only when the maximum rose by more than 2^kDefer somewhere
    if (__ballot(mx > m + kDefer) != 0) {
      mx = fmaxf(mx, xor16(mx));
      mx = fmaxf(mx, xor32(mx));
      const float mn = fmaxf(m, mx);
      const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      if (i) {
        l *= al;
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] *= al;
      }
    }
    float back;
    const float lw = value_weight(vs, vs / vref, back) + (m == -INFINITY ? kBias : kBias - m);
    h8 pa[2];
    float ls = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {                       // (a poisoned page: NaN, as for its whole row)
      const float p = __builtin_amdgcn_exp2f(fmaf(sc[e], f, lw));
      ls += p;
      pa[e >> 3][e & 7] = (_Float16)p;
    }
    l += ls * back;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h8<FP8>(vr[n].x, vr[n].y), pa[0], o[n], 0, 0, 0);
      o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h8<FP8>(vr[n].z, vr[n].w), pa[1], o[n], 0, 0, 0);
    }
    if (more) load_values(i + 1);
  }
  l += xor16(l);
  l += xor32(l);

  // merge the waves: lane (head pr, kg) holds dims 16 n + 4 kg + 0..3 of its head
  __shared__ float wm[NW][16], wl[NW][16];
  __shared__ __align__(16) float wo[NW][16][D + 4];
  if (kg == 0) { wm[wave][pr] = m; wl[wave][pr] = l; }
  if (pr < gn) {
#pragma unroll
    for (int n = 0; n < ND; ++n) *reinterpret_cast<f4*>(&wo[wave][pr][16 * n + 4 * kg]) = o[n] * vref;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gn * (D / 4); i += 64 * NW) {
    const int g = i / (D / 4), d = 4 * (i % (D / 4));
    float M = wm[0][g];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, wm[w][g]);
    float L = 0.f;
    f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = wm[w][g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wm[w][g] - M);
      // a wave whose l is NaN saw a poisoned page: its maximum may still be -inf
      const float lw = wl[w][g];
      L += lw != lw ? lw : lw * e;
      if (e != 0.f) y += *reinterpret_cast<f4*>(&wo[w][g][d]) * e;
    }
    const int h = kh * a.G + h0 + g;
    if (a.parts > 1) {
      const long row = ((long)part * a.sg.N + t) * a.H + h;
      *reinterpret_cast<f4*>(a.po + row * D + d) = y;
      if (d == 0) { a.pml[2 * row] = M; a.pml[2 * row + 1] = L; }
    } else {
      y *= L == 0.f ? 0.f : 1.f / L;
      if (a.x8) put_q8<4>(a, t, (long)h * D + d, {y[0], y[1], y[2], y[3]});
      if (!a.out) continue;
      uint16_t* at = static_cast<uint16_t*>(a.out) + (long)t * a.so_tok + (long)h * a.so_head + d;
      const uint32_t w0 = Elem<T>::put(y[0]) | (uint32_t)Elem<T>::put(y[1]) << 16;
      const uint32_t w1 = Elem<T>::put(y[2]) | (uint32_t)Elem<T>::put(y[3]) << 16;
      if (a.wide_o) {
        *reinterpret_cast<uint2*>(at) = make_uint2(w0, w1);
      } else {
        at[0] = (uint16_t)w0; at[1] = (uint16_t)(w0 >> 16); at[2] = (uint16_t)w1; at[3] = (uint16_t)(w1 >> 16);
      }
    }
  }
}

// Joins the partials of one (row, head): NW waves take every NW'th partial, a lane D / 64 dims.  Every
// partial's maximum and sum are written, also an empty one's (-inf, 0), whose output is not: all loads
// go out at once and an empty one's weight is 0.
template <int D, int T, int NW, bool DECODE>
__global__ void __launch_bounds__(64 * NW) kv8_join_kernel(const AttnArgs a) {
  constexpr int E = D / 64, B = 8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x, t = blockIdx.y, np = a.parts;
  if (!DECODE) {
    Row at;
    if (!find_row(a.sg, t, at)) return;                  // no partials: the output row stays
  }
  const long row = (long)t * a.H + h, step = (long)a.sg.N * a.H;
  float M = -INFINITY, L = 0.f;
  float y[E];
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = 0.f;
  for (int b = 0; b < np; b += 64) {                     // lane = partial
    const int n = min(64, np - b);
    float x[B][E];
    auto load = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const float* src = a.po + (row + (long)(b + min(i + NW * u, n - 1)) * step) * D + E * lane;
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = src[e];
      }
    };
    const long at = row + (long)(b + min(lane, n - 1)) * step;
    float pm = a.pml[2 * at], pl = a.pml[2 * at + 1];
    load(wave);
    if (lane >= n) { pm = -INFINITY; pl = 0.f; }
    const float mn = fmaxf(M, wave_max(pm));
    const float al = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
    const float w = pm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm - mn);
    L = L * al + wave_sum(pl != pl ? pl : pl * w);
    M = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] *= al;
    for (int i = wave; i < n; i += NW * B) {             // B partials in flight
      if (i != wave) load(i);
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int p = min(i + NW * u, n - 1);
        const float ww = i + NW * u < n ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), p)) : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = ww != 0.f ? __fmaf_rn(ww, x[u][e], y[e]) : y[e];
      }
    }
  }
  if constexpr (NW > 1) {
    __shared__ float part[NW][D];
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][E * lane + e] = y[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < NW; ++w)
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] += part[w][E * lane + e];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] *= inv;
  if (a.out) {
    uint16_t* at = static_cast<uint16_t*>(a.out) + (long)t * a.so_tok + (long)h * a.so_head + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) at[e] = Elem<T>::put(y[e]);
  }
  if constexpr (DECODE) {
    if (a.x8) put_q8<E>(a, t, (long)h * D + E * lane, y);
  }
}

// ---------------------------------------------------------------- prompt attention
// Rows of one KV head are token-major, row = token x G + head in group; a workgroup has RW waves of 32
// rows, or two slots of RW waves that take the row block's pages in turn, each through its own buffers,
// and add up in LDS at the end (for grids too small to give a SIMD two waves otherwise: the chain of
// pages halves, 1024 rows at 0 31 -> 26 us).  Each page goes through LDS once for all rows, turned to
// fp16 on the way (double buffered; the next page's loads are in flight during this one's maths).
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16, a lane owns one query row: softmax and
// rescaling need one exchange (lane ^ 32).  The key of position p lies in LDS row p with bits 2 and 3
// swapped, so that the score registers of a lane are, in order, the P operand's consecutive positions: P
// never moves.
// What bounds it: matrix and vector instructions of a SIMD's two waves hardly overlap as they are scheduled
// here (8192 rows at 0: matrix cores busy 40 % of the time, vector units 46 %): both waves leave a page's
// barrier at once and ask for the same unit in the same order.  Half of the vector time is the exponents;
// three waves a SIMD took 12 % fewer cycles at a clock 11 % lower.  Waves half a page apart were not tried.
// 8192 at 0 503 to 513 us, 950 TFLOP/s of visible pairs (a library product of two 8192 matrices reaches
// 1450); 512 at 31488 252 to 256 us, its 224 workgroups on 256 CUs.  Tried and not taken, by the form that
// took 496 us: 64 rows a wave (twice the registers, one wave a SIMD: 660 us), the next page's scores ahead of
// this page's weights (580), pages turned to fp16 images in memory once and loaded into LDS directly (503,
// and 284 for 512 at 31488), wave priorities (no change).
__device__ __forceinline__ int swap23(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

// A tile's LDS image: key rows of 2 D bytes and value rows of 128 (64 positions of a dim) in fp16, each
// row 16 bytes longer than its data, so that rows lie in banks of their own and a lane's fragments are
// constants behind one address.  A key row has its even 16-byte chunks first (a thread stages chunks 2 c
// and 2 c + 1: the next thread's do not meet them).
template <int D>
struct Image {
  static constexpr int kKeyRow = 2 * D + 16, kValueRow = 2 * kPage + 16;
  static constexpr int kKeys = kPage * kKeyRow, kValues = D * kValueRow;    // bytes, multiples of 1024
  static __device__ __forceinline__ int key(int row, int ch) {
    return row * kKeyRow + 16 * (ch >> 1 | (ch & 1) * (D / 16));
  }
  static __device__ __forceinline__ int value(int d, int ch) { return d * kValueRow + 16 * ch; }
};

// 16 key codes (chunk c of the page's) / 16 value codes into the image
template <int D, bool FP8>
__device__ __forceinline__ void image_keys(char* to, int c, const uint4& w) {
  const int row = swap23(c / (D / 16)), ch = 2 * (c % (D / 16));
  *reinterpret_cast<h8*>(to + Image<D>::key(row, ch)) = codes_h8<FP8>(w.x, w.y);
  *reinterpret_cast<h8*>(to + Image<D>::key(row, ch + 1)) = codes_h8<FP8>(w.z, w.w);
}
// codes of positions that were never written (`live` and up of the page's 64) may be NaN, and a weight of
// 0 would not hide them
template <int D, bool FP8>
__device__ __forceinline__ void image_values(char* to, int c, const uint4& v, int live) {
  const int d = c >> 2, ch = 2 * (c & 3);
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (FP8 && live < kPage) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (8 * ch + e >= live) w[e >> 2] &= ~(0xffu << (8 * (e & 3)));
  }
  *reinterpret_cast<h8*>(to + Image<D>::value(d, ch)) = codes_h8<FP8>(w[0], w[1]);
  *reinterpret_cast<h8*>(to + Image<D>::value(d, ch + 1)) = codes_h8<FP8>(w[2], w[3]);
}

template <int D, bool FP8, int T, int RW, int SLOTS>
__global__ void __launch_bounds__(64 * RW * SLOTS, 2) kv8_prompt_kernel(const AttnArgs a) {
  typedef Image<D> I;
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int NT = 64 * RW, NCH = kPage * D / 16, CH = (NCH + NT - 1) / NT;   // 16-code chunks a thread
  constexpr int BUF = I::kKeys + I::kValues;
  __shared__ __align__(16) char shared[SLOTS * 2 * BUF];
  const int slot = SLOTS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  const int tid = threadIdx.x - slot * NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* lds = shared + slot * 2 * BUF;
  const int r = lane & 31, hh = lane >> 5;
  const int kh = blockIdx.x % a.c.Hkv;
  // later pieces (of a causal prompt: the longest) first
  const int unit = a.units - 1 - (int)(blockIdx.x / a.c.Hkv);
  Piece pc;
  if (!find_piece(a.sg, unit, [&](int n, int) { return (int)(((long)n * a.G + 32 * RW - 1) / (32 * RW)); }, pc))
    return;
  const int s = pc.s, row0 = pc.row, cnt = pc.cnt, start = pc.pos;
  const int rows = cnt * a.G, R0 = pc.index * 32 * RW;
  const int span = min(a.span, a.c.width * kPage);
  const int t_hi = min(cnt - 1, (R0 + 32 * RW - 1) / a.G);
  const Seen seen = seen_pages(start + R0 / a.G, start + t_hi, span, a.window, a.sinks);
  const int each = (seen.n + a.parts - 1) / a.parts;
  const int t0 = min(seen.n, (int)blockIdx.y * each), t1 = min(seen.n, t0 + each);
  // this lane's row
  const int rr = R0 + wave * 32 + r;
  const bool valid = rr < rows;
  const int tok = valid ? rr / a.G : cnt - 1;
  const int head = kh * a.G + (valid ? rr - tok * a.G : 0);
  const int pos = start + tok;
  // this wave's positions
  const bool wave_in = R0 + wave * 32 < rows;
  const int w_lo = start + min(cnt - 1, (R0 + wave * 32) / a.G);
  const int w_hi = start + min(cnt - 1, (R0 + wave * 32 + 31) / a.G);
  const int end = min(start + cnt, span);                // keys behind it were never written

  h8 qa[KS];
  float qf = a.c2;
  {
    const uint16_t* qr = a.q + (long)(row0 + tok) * a.sq_tok + (long)head * a.sq_head;
    float x[KS][8], amax = 0.f;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      load_n<T, 8>(qr + 16 * st + 8 * hh, a.wide_q, x[st]);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[st][e]));
    }
    float f = 1.f;
    if constexpr (T == kBF16) {
      amax = fmaxf(amax, xor32(amax));
      f = fit_f16(amax);
      qf /= f;
    }
    f *= a.sign;
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) qa[st][e] = (_Float16)(x[st][e] * f);
  }
  float m = -INFINITY, l = 0.f, vref = 0.f;
  f16v o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;

  uint4 kr[CH], vr[CH];
  auto load_tile = [&](int id) __attribute__((always_inline)) {
    const long at = ((long)max(id, 0) * a.c.Hkv + kh) * kPage * D;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int c = tid + u * NT;
      if (NCH % NT == 0 || c < NCH) {
        kr[u] = reinterpret_cast<const uint4*>(a.c.k + at)[c];
        vr[u] = reinterpret_cast<const uint4*>(a.c.v + at)[c];
      }
    }
  };
  auto store_tile = [&](int buf, int live) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int c = tid + u * NT;
      if (NCH % NT == 0 || c < NCH) {
        image_keys<D, FP8>(lds + buf * BUF, c, kr[u]);
        image_values<D, FP8>(lds + buf * BUF + I::kKeys, c, vr[u], live);
      }
    }
  };
  // Table entries and scales of 64 pages at a time, a page a lane: a load for every page would have to be
  // waited for with the tile's own loads, which are in the same queue.
  int held = t0 - 64, my_id = -1;
  float my_ks = 0.f, my_vs = 0.f;
  auto entry = [&](int t, int& id, float& ks, float& vs) __attribute__((always_inline)) {
    if (t >= held + 64) {                                // uniform; t only grows
      held = t;
      my_id = -1;
      if (t + lane < t1) {
        my_id = a.c.page(s, seen.page(t + lane));
        const long sc = (long)max(my_id, 0) * a.c.Hkv + kh;
        my_ks = a.c.ks[sc];
        my_vs = a.c.vs[sc];
      }
    }
    id = __builtin_amdgcn_readlane(my_id, t - held);
    ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_ks), t - held));
    vs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_vs), t - held));
  };
  const int kfrag = I::key(r, hh), vfrag = I::kKeys + I::value(r, hh);

  int id = -1;
  float ks = 0.f, vs = 0.f;
  int t = t0 + slot;
  if (t < t1) {
    entry(t, id, ks, vs);
    load_tile(id);
    store_tile(0, end - seen.page(t) * kPage);
  }
  __syncthreads();
  for (int buf = 0; t < t1 + slot; t += SLOTS, buf ^= 1) {   // (as many turns in every slot)
    const int base = seen.page(t) * kPage;
    int id1 = -1;
    float ks1 = 0.f, vs1 = 0.f;
    if (t + SLOTS < t1) {
      entry(t + SLOTS, id1, ks1, vs1);
      load_tile(id1);
    }
    const bool hidden = base > w_hi || (a.window > 0 && base + kPage - 1 <= w_lo - a.window && base >= a.sinks);
    if (wave_in && id >= 0 && !hidden) {                 // (id is -1 behind t1)
      // The reference scale is the row's own: its neighbours may see other pages, and weights relative to a
      // larger scale that only those see would be lost.  Ahead of the matrix instructions, which hide most of
      // it (8192 at 0 497 us with one reference for the wave, 503 so, 531 behind the masks), and by the
      // reciprocal, exact for powers of two (508 with a division).
      const bool poisoned = ks != ks || vs != vs;
      const int top = min(min(pos, end - 1), base + kPage - 1);             // the row's last key of the page
      const bool sees = top >= base && (a.window <= 0 || top > pos - a.window || base < a.sinks);
      const float own = sees && !poisoned ? vs : 0.f;
      if (__ballot(own > vref) != 0) {
        const float q = own > vref ? vref / own : 1.f;
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] *= q;
        vref = fmaxf(vref, own);
      }
      float back;
      const float vw = value_weight(own, own * __builtin_amdgcn_rcpf(vref), back);
      const char* kl = lds + buf * BUF + kfrag;
      f16v sc[2];
      const f16v zero = {};
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              *reinterpret_cast<const h8*>(kl + 16 * st + 32 * b * I::kKeyRow), qa[st], st ? sc[b] : zero, 0, 0, 0);
      // the order: two key fragments of either half read ahead of the matrix instructions that take them
      constexpr int AHEAD = 2;
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);            // LDS reads
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        if (st + AHEAD < KS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);                  // matrix instructions
      }
      const float f = score_factor(poisoned ? 0.f : ks, qf);
      const bool whole = base + kPage - 1 <= w_lo && base + kPage <= end &&
                         (a.window <= 0 || base > w_hi - a.window || base + kPage <= a.sinks);
      if (!whole) {
        const int at = base + 8 * hh, hi = min(pos, end - 1) - at;          // of the registers' own offsets
        const int lo = (a.window > 0 ? pos - a.window : -1) - at, sinks = a.sinks - at;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int x = 32 * b + 16 * (i >> 3) + (i & 7);
            sc[b][i] = ((x <= hi) & ((x > lo) | (x < sinks))) ? sc[b][i] : -INFINITY;
          }
      }
      float mx = sc[0][0];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[b][i]);
      mx *= f;
      if (__ballot(mx > m + kDefer) != 0) {
        mx = fmaxf(mx, xor32(mx));
        const float mn = fmaxf(m, mx);
        const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] *= al;
      }
      const float up = m == -INFINITY ? kBias : kBias - m;
      if (poisoned) {                                    // NaN for the rows that see a key of it
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[b][i] = sc[b][i] == -INFINITY ? sc[b][i] : __builtin_nanf("");
      }
      if (vw < -6.f) {                                   // fp16 weights of so small values would lose their sum
        back = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(fmaf(sc[b][i], f, up));
      }
      // The row's sum is one of the weights as they were rounded, in 32 bits: what rounding does to a weight
      // then stands above and below the line.  With the unrounded weights, at the same speed, errors were up
      // to 8 % larger (rms; 6 x 300: 1.14e-4 -> 1.22e-4 of outputs of 0.42) and a third at the worst.
      h8 pa[4];
      const h2 one = {(_Float16)1.f, (_Float16)1.f};
      float ls0 = 0.f, ls1 = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const h2 p = {(_Float16)__builtin_amdgcn_exp2f(fmaf(sc[b][i], f, vw + up)),
                        (_Float16)__builtin_amdgcn_exp2f(fmaf(sc[b][i + 1], f, vw + up))};
          float& ls = i & 2 ? ls1 : ls0;
          ls = __builtin_amdgcn_fdot2(p, one, ls, false);
          pa[2 * b + (i >> 3)][i & 7] = p[0];
          pa[2 * b + (i >> 3)][(i & 7) + 1] = p[1];
        }
      l = fmaf(ls0 + ls1, back, l);
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int b = 0; b < DB; ++b)
          o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              *reinterpret_cast<const h8*>(lds + buf * BUF + vfrag + 32 * st + 32 * b * I::kValueRow), pa[st], o[b],
              0, 0, 0);
    }
    if (t + SLOTS < t1) store_tile(buf ^ 1, end - seen.page(t + SLOTS) * kPage);
    id = id1; ks = ks1; vs = vs1;
    __syncthreads();
  }
  l += xor32(l);
  if constexpr (SLOTS == 2) {                            // the second slot's share joins the first's
    float* to = reinterpret_cast<float*>(shared) + wave * (16 * DB + 2) * 64 + lane;
    if (slot) {
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) to[64 * (16 * b + i)] = o[b][i] * vref;
      to[64 * 16 * DB] = m;
      to[64 * (16 * DB + 1)] = l;
    }
    __syncthreads();
    if (slot) return;
    const float m2 = to[64 * 16 * DB], l2 = to[64 * (16 * DB + 1)], M = fmaxf(m, m2);
    const float e1 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    const float e2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - M);
    // (a NaN sum: a poisoned page, whose maximum may still be -inf)
    l = (l != l ? l : l * e1) + (l2 != l2 ? l2 : l2 * e2);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = o[b][i] * vref * e1 + to[64 * (16 * b + i)] * e2;
    m = M;
    vref = 1.f;
  }
  if (!valid) return;
  const long grow = (long)row0 + tok;
  if (a.parts > 1) {
    const long prow = ((long)blockIdx.y * a.sg.N + grow) * a.H + head;
    float* at = a.po + prow * D;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f4*>(at + 32 * b + 2 * i + 4 * hh) =
            f4{o[b][i] * vref, o[b][i + 1] * vref, o[b][i + 2] * vref, o[b][i + 3] * vref};
    if (hh == 0) { a.pml[2 * prow] = m; a.pml[2 * prow + 1] = l; }
    return;
  }
  const float inv = l == 0.f ? 0.f : vref / l;
  uint16_t* at = static_cast<uint16_t*>(a.out) + grow * a.so_tok + (long)head * a.so_head;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint16_t* w = at + 32 * b + 2 * i + 4 * hh;
      const uint32_t w0 = Elem<T>::put(o[b][i] * inv) | (uint32_t)Elem<T>::put(o[b][i + 1] * inv) << 16;
      const uint32_t w1 = Elem<T>::put(o[b][i + 2] * inv) | (uint32_t)Elem<T>::put(o[b][i + 3] * inv) << 16;
      if (a.wide_o) {
        *reinterpret_cast<uint2*>(w) = make_uint2(w0, w1);
      } else {
        w[0] = (uint16_t)w0; w[1] = (uint16_t)(w0 >> 16); w[2] = (uint16_t)w1; w[3] = (uint16_t)(w1 >> 16);
      }
    }
}

}  // namespace

// ---------------------------------------------------------------- C entries
// A call is one record of 64-bit fields (addresses, sizes and strides in elements), in the order of
// these structs: passing some thirty arguments one by one cost the caller more than the kernel runs.
namespace {

struct PoolCall {
  int64_t k, v, ks, vs, table, pool, hkv, d, fp8, width, stride;
};
struct RowsCall {
  int64_t at, tok, head;               // address, row and head stride
};
struct AppendCall {
  PoolCall c;
  int64_t start, cu, s, n;
  RowsCall k, v, q, qo;                // q, qo: address 0 for none
  int64_t heads, cos_t, sin_t, table_rows, type, otype;   // types: 0 fp16, 1 bf16, 2 fp32; cos_t 0: no rotation
};
struct ReadCall {
  PoolCall c;
  int64_t start, cu, s, n;
  RowsCall k, v;
  int64_t type;
};
struct AttnCall {
  PoolCall c;
  int64_t start, cu, s, n;             // decode: start = positions, cu unused, n = s
  RowsCall q, out;                     // out: address 0 for none (decode with x8)
  int64_t heads, span, window, sinks, type;
  int64_t x8, dx, sx;                  // decode: Q8 output or 0
};

template <typename T>
T* ptr(int64_t a) {
  return reinterpret_cast<T*>(a);
}
bool wide16(const RowsCall& r, long esize) {
  return (r.at & 15) == 0 && (r.tok * esize) % 16 == 0 && (r.head * esize) % 16 == 0;
}
int launched() { return hipGetLastError() == hipSuccess ? 0 : 1; }
bool in(int64_t x, int64_t low, int64_t high) { return x >= low && x <= high; }

// D and the code type to template arguments
template <typename F>
int by_format(const PoolCall& c, F f) {
  using I64 = std::integral_constant<int, 64>;
  using I128 = std::integral_constant<int, 128>;
  if (c.d == 128) return c.fp8 ? f(I128{}, std::true_type{}) : f(I128{}, std::false_type{});
  if (c.d == 64) return c.fp8 ? f(I64{}, std::true_type{}) : f(I64{}, std::false_type{});
  return 2;
}

bool good_pool(const PoolCall& c) {
  return c.k && c.v && c.ks && c.vs && c.table && ((c.k | c.v) & 15) == 0 && in(c.pool, 1, 0x7fffffff) &&
         in(c.hkv, 1, 65535) && in(c.width, 1, 1 << 24) && in(c.stride, 0, 0x7fffffff);
}
bool good_segs(int64_t start, int64_t cu, int64_t s, int64_t n) {
  return start && cu && in(s, 1, 0x3fffffff) && in(n, 1, 0x3fffffff);
}
Pool make_pool(const PoolCall& c) {
  return Pool{ptr<uint8_t>(c.k), ptr<uint8_t>(c.v), ptr<float>(c.ks), ptr<float>(c.vs), ptr<const int>(c.table),
              (int)c.pool, (int)c.hkv, (int)c.width, (int)c.stride};
}
Segs make_segs(int64_t start, int64_t cu, int64_t s, int64_t n) {
  return Segs{ptr<const int>(start), ptr<const int>(cu), (int)s, (int)n};
}
bool good_attn(const AttnCall& c) {
  return good_pool(c.c) && c.start && c.q.at && in(c.heads, 1, 0x3fffffff) && c.heads % c.c.hkv == 0 &&
         in(c.type, 0, 1) && in(c.span, 1, c.c.width * kPage) && in(c.window, 0, 1 << 30) && in(c.sinks, 0, 1 << 30);
}
bool good_decode(const AttnCall& c) { return good_attn(c) && in(c.s, 1, 65535) && c.n == c.s; }
bool good_prompt(const AttnCall& c) {
  return good_attn(c) && good_segs(c.start, c.cu, c.s, c.n) && c.n * (c.heads / c.c.hkv) <= 0x3fffffffL;
}
long work_floats_of(const AttnCall& c, long parts) { return parts == 1 ? 0 : parts * c.n * c.heads * (c.c.d + 2); }
AttnArgs make_attn(const AttnCall& c, float scale, void* work, long parts) {
  AttnArgs a{};
  a.c = make_pool(c.c);
  a.sg = make_segs(c.start, c.cu, c.s, c.n);
  a.q = ptr<const uint16_t>(c.q.at);
  a.out = ptr<void>(c.out.at);
  a.po = static_cast<float*>(work);
  a.pml = work ? a.po + parts * c.n * c.heads * c.c.d : nullptr;
  a.x8 = ptr<int8_t>(c.x8);
  a.dx = ptr<float>(c.dx);
  a.sx = ptr<float>(c.sx);
  a.sq_tok = c.q.tok; a.sq_head = c.q.head; a.so_tok = c.out.tok; a.so_head = c.out.head;
  a.H = (int)c.heads; a.G = (int)(c.heads / c.c.hkv); a.D = (int)c.c.d;
  a.span = (int)c.span; a.window = (int)c.window; a.sinks = (int)c.sinks; a.parts = (int)parts;
  a.c2 = (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  a.sign = scale < 0.f ? -1.f : 1.f;
  a.wide_q = wide16(c.q, 2);
  a.wide_o = c.out.at && wide16(c.out, 2);
  return a;
}

// most pages that queries at `rows` neighbouring positions see
long most_seen(const AttnCall& c, long rows) {
  const long n = (c.span + kPage - 1) / kPage;
  if (c.window <= 0) return n;
  const long w = (c.window + rows + 61) / kPage + 1 + (c.sinks + kPage - 1) / kPage;
  return w < n ? w : n;
}

struct DecodePlan {
  int nw, per;
  long parts;
};
// Workgroups that share a row's pages: as many as let all of them run in one round, 512 of 4 waves, two on
// each CU (8 x 32768 44 us; at most 384 49; 576 and more, a second round, 48; 32 x 16000 in 4 parts 98, in
// 5 112).  At most 64, past which the join costs what the shorter chains save (1 x 32768 in 64 parts 13.9,
// in 128 16.0), unless a wave would have more than the 64 pages whose table entries it holds.  Where one
// part fills the CUs, a wave has 4 pages before there is a second one (64 x 1000 in one part 14.7, in two
// 18.5); where it does not, one page is enough (1 x 4000 with one page a wave 9.1, with two 10.7).
// Waves that would have two pages or more go 8 to a workgroup and half as many parts, if those fill three
// quarters of the CUs: fewer partials (32 x 16000 with a window 57 -> 51, 64 x 4000 49 -> 45, 48 x 2000
// 25 -> 20; with 160 of 256 CUs 60 -> 61; with one page a wave 9.2 -> 10.8).  Those figures are of pages in
// random order.  Where a row's pages follow one another and rows start at multiples of 2 MB, so that all parts
// stream in step, 8 waves are the slower ones: 8 x 32000 54 to 62 us, 4 waves 50, in random order 50 and 49.
// Up to 8 pages run in one workgroup of 8 waves, which needs no join: 500 positions 8.1 us against 9.2.
// (A row's sums therefore depend, in their last bits, on how many rows and what span are beside it.)
DecodePlan decode_plan(const AttnCall& c) {
  const long n = most_seen(c, 1);
  if (n <= 8) return {8, 1, 1};
  const long chains = c.s * c.c.hkv * ((c.heads / c.c.hkv + 15) / 16);
  auto plan = [&](int nw, long grid) -> DecodePlan {
    const long fill = grid / chains, few = chains >= grid / 2 ? 16 / nw : 1;
    const long worth = (n + nw * few - 1) / (nw * few), need = (n + 64 * nw - 1) / (64 * nw);
    long parts = fill > 64 ? 64 : fill;
    parts = parts > worth ? worth : parts;
    parts = parts < need ? need : parts;
    const long per = (n + nw * parts - 1) / (nw * parts);
    return {nw, (int)per, (n + nw * per - 1) / (nw * per)};
  };
  const DecodePlan four = plan(4, 512);
  return four.per > 1 && chains <= 256 && 256 / chains * chains >= 192 ? plan(8, 256) : four;
}

struct PromptPlan {
  int rw, slots;                       // waves of 32 rows, key slots
  long units, parts;
};
// The workgroup's form and how many workgroups share a row block's pages, by what they take (microseconds,
// measured at D 128, and taken for D 64 too: there the choice is the best form or within 4 % of it for 6 x 300
// at 700, 128 to 2048 rows at 0, 512 at 512 and at 16000, and 9 % off at 4096 rows): its start and end, partly hidden in rounds after the first; a page, 1.5 for 4 waves
// alone on their CU and 2.05 beside another workgroup (two fit), 1.95 for 8 waves of rows, 1.1 for 4 of
// rows in two key slots (of either one fits); partial outputs cost a join launch and their bytes.  The
// time is the longest row block's or that of the rounds over the chip, whichever is more; a causal chunk's
// own pages count half, as its row blocks see them on average.
// The three forms without parts: 128 rows at 0 10.5, 13.8, 11.3 us; 512 at 512 30, 38, 26; 2048 at 0 58,
// 68, 50; 4096 at 0 145, 133, 155; 6 x 300 at 700 36, 39, 41.  Parts: 16 rows at 500 in 1 part 20, in 8
// 13; 512 rows at 0 in 1 part 19, in 2 28; 512 at 16000, 8 waves, in 1, 2, 4, 8 parts 458, 247, 138, 151.
PromptPlan prompt_plan(const AttnCall& c) {
  struct Form {
    int rw, slots, fit;                // fit: workgroups on the chip
    double base, again, page;
  };
  constexpr Form forms[] = {{4, 1, 512, 7.2, 2.5, 1.5}, {8, 1, 256, 9, 3.5, 1.95}, {4, 2, 256, 8.4, 6, 1.1}};
  const long G = c.heads / c.c.hkv;
  PromptPlan best{4, 1, 0, 1};
  double least = 0;
  for (const Form& f : forms) {
    const long rows = 32 * f.rw;
    long units = c.n * G / rows + c.s;
    if (G <= rows && units > c.n) units = c.n;
    const long n = most_seen(c, (rows + G - 1) / G + 1);
    const long own = c.n / (kPage * c.s);
    const double mean = n - 0.5 * (own < n ? own : n);
    const double bytes = 8.0 * c.n * c.heads * c.c.d;
    for (long p = 1; p <= n && p <= (c.n > 65535 ? 1 : 64); ++p) {   // (the join's grid has 16 bits of rows)
      const double join = p > 1 ? 4.5 + p * bytes / 4.5e6 : 0;
      if (best.units && f.base + join > least) break;
      const long wgs = units * c.c.hkv * p, rounds = (wgs + f.fit - 1) / f.fit;
      const double crowd = (wgs * mean / n - 256) / 128;  // CUs with two workgroups: none to most
      const double page = f.page + (f.fit == 512 ? 0.55 * (crowd < 0 ? 0 : crowd > 1 ? 1 : crowd) : 0);
      const double longest = (double)((n + p - 1) / p) * page, all = rounds * mean / p * page;
      const double t = f.base + f.again * (rounds - 1) + (longest > all ? longest : all) + join;
      if (best.units == 0 || t < least) {
        least = t;
        best = {f.rw, f.slots, units, p};
      }
    }
  }
  return best;
}

}  // namespace

extern "C" {

int amdk8s_llm_kv8_page() { return kPage; }

// Each entry returns 0: launched, 1: a launch error, 2: a bad argument.

// Rows of k / v (and q) of the segments into the cache.
int amdk8s_llm_kv8_append(const void* call, void* stream) {
  const AppendCall& c = *static_cast<const AppendCall*>(call);
  if (!good_pool(c.c) || !good_segs(c.start, c.cu, c.s, c.n) || !c.k.at || !c.v.at) return 2;
  if (!c.q.at != !c.qo.at || (c.q.at && !in(c.heads, 1, 0x3fffffff)) || !c.cos_t != !c.sin_t) return 2;
  if (!in(c.type, 0, 2) || !in(c.otype, 0, 1) || (c.type < 2 && c.otype != c.type)) return 2;
  if (c.cos_t && (!in(c.table_rows, c.c.width * kPage, 0x7fffffff) || ((c.cos_t | c.sin_t) & 15))) return 2;
  AppendArgs a{};
  a.c = make_pool(c.c);
  a.sg = make_segs(c.start, c.cu, c.s, c.n);
  a.k = ptr<void>(c.k.at); a.v = ptr<void>(c.v.at); a.q = ptr<void>(c.q.at); a.qo = ptr<void>(c.qo.at);
  a.cos_t = ptr<const float>(c.cos_t);
  a.sin_t = ptr<const float>(c.sin_t);
  a.sk_tok = c.k.tok; a.sk_head = c.k.head; a.sv_tok = c.v.tok; a.sv_head = c.v.head;
  a.sq_tok = c.q.tok; a.sq_head = c.q.head; a.so_tok = c.qo.tok; a.so_head = c.qo.head;
  a.H = (int)c.heads;
  const int es = c.type == kF32 ? 4 : 2;
  a.wide_kv = wide16(c.k, es) && wide16(c.v, es);
  a.wide_q = c.q.at && wide16(c.q, es) && wide16(c.qo, 2);
  a.table_rows = c.cos_t ? (int)c.table_rows : 0x7fffffff;
  // query rows a wave: one until the waves fill the chip, then up to four (the search for a row's segment
  // and its table rows are paid once a wave)
  a.per = c.n >= 16384 ? 4 : c.n >= 8192 ? 2 : 1;
  const long units = most_pages(c.n, c.s), qb = c.q.at ? (c.n + 4 * a.per - 1) / (4 * a.per) : 0;
  if (units * c.c.hkv + qb > 0x7fffffffL) return 2;
  a.units = (int)units;
  const dim3 grid((unsigned)(units * c.c.hkv + qb));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_format(c.c, [&](auto d, auto f) -> int {
    constexpr int DD = decltype(d)::value;
    constexpr bool F8 = decltype(f)::value;
    if (c.type == kF16) hipLaunchKernelGGL((kv8_append_kernel<DD, F8, kF16, kF16>), grid, dim3(256), 0, st, a);
    else if (c.type == kBF16) hipLaunchKernelGGL((kv8_append_kernel<DD, F8, kBF16, kBF16>), grid, dim3(256), 0, st, a);
    else if (c.otype == kF16) hipLaunchKernelGGL((kv8_append_kernel<DD, F8, kF32, kF16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_append_kernel<DD, F8, kF32, kBF16>), grid, dim3(256), 0, st, a);
    return launched();
  });
}

// Cached positions of the segments as values.
int amdk8s_llm_kv8_read(const void* call, void* stream) {
  const ReadCall& c = *static_cast<const ReadCall*>(call);
  if (!good_pool(c.c) || !good_segs(c.start, c.cu, c.s, c.n) || !c.k.at || !c.v.at || !in(c.type, 0, 2)) return 2;
  ReadArgs a{};
  a.c = make_pool(c.c);
  a.sg = make_segs(c.start, c.cu, c.s, c.n);
  a.ko = ptr<void>(c.k.at); a.vo = ptr<void>(c.v.at);
  a.sk_tok = c.k.tok; a.sk_head = c.k.head; a.sv_tok = c.v.tok; a.sv_head = c.v.head;
  const int es = c.type == kF32 ? 4 : 2;
  a.wide = wide16(c.k, es) && wide16(c.v, es);
  const long blocks = most_pages(c.n, c.s) * c.c.hkv;
  if (blocks > 0x7fffffffL) return 2;
  const dim3 grid((unsigned)blocks);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_format(c.c, [&](auto d, auto f) -> int {
    constexpr int DD = decltype(d)::value;
    constexpr bool F8 = decltype(f)::value;
    if (c.type == kF16) hipLaunchKernelGGL((kv8_read_kernel<DD, F8, kF16>), grid, dim3(256), 0, st, a);
    else if (c.type == kBF16) hipLaunchKernelGGL((kv8_read_kernel<DD, F8, kBF16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_read_kernel<DD, F8, kF32>), grid, dim3(256), 0, st, a);
    return launched();
  });
}

// fp32 workspace (in floats) of the call: 0 when its partials need no join, -1 for a bad argument
long amdk8s_llm_kv8_decode_work(const void* call) {
  const AttnCall& c = *static_cast<const AttnCall*>(call);
  return good_decode(c) ? work_floats_of(c, decode_plan(c).parts) : -1;
}

// One query row a sequence at position start[s] (-1: nothing to see, zeros); keys at or behind `span` are
// not attended.
int amdk8s_llm_kv8_decode(const void* call, float scale, void* work, long work_floats, void* stream) {
  const AttnCall& c = *static_cast<const AttnCall*>(call);
  if (!good_decode(c) || (!c.out.at && !c.x8) || (c.x8 && (!c.dx || !c.sx))) return 2;
  const DecodePlan plan = decode_plan(c);
  const long need = work_floats_of(c, plan.parts);
  if (need > work_floats || (need && (!work || ((uintptr_t)work & 15)))) return 2;
  if (plan.parts > 65535) return 2;
  AttnArgs a = make_attn(c, scale, need ? work : nullptr, plan.parts);
  a.per = plan.per;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(c.c.hkv * ((a.G + 15) / 16)), (unsigned)plan.parts, (unsigned)c.s);
  return by_format(c.c, [&](auto d, auto f) -> int {
    constexpr int DD = decltype(d)::value;
    constexpr bool F8 = decltype(f)::value;
    auto go = [&](auto nw, auto once) {
      constexpr int NW = decltype(nw)::value;
      constexpr bool ON = decltype(once)::value;
      if (c.type == kF16) hipLaunchKernelGGL((kv8_decode_kernel<DD, F8, kF16, NW, ON>), grid, dim3(64 * NW), 0, st, a);
      else hipLaunchKernelGGL((kv8_decode_kernel<DD, F8, kBF16, NW, ON>), grid, dim3(64 * NW), 0, st, a);
    };
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    if (a.G > 16) plan.nw == 8 ? go(I8{}, std::false_type{}) : go(I4{}, std::false_type{});
    else plan.nw == 8 ? go(I8{}, std::true_type{}) : go(I4{}, std::true_type{});
    if (need) {
      const dim3 rows((unsigned)c.heads, (unsigned)c.s);
      if (c.type == kF16) hipLaunchKernelGGL((kv8_join_kernel<DD, kF16, 4, true>), rows, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((kv8_join_kernel<DD, kBF16, 4, true>), rows, dim3(256), 0, st, a);
    }
    return launched();
  });
}

long amdk8s_llm_kv8_prompt_work(const void* call) {
  const AttnCall& c = *static_cast<const AttnCall*>(call);
  return good_prompt(c) ? work_floats_of(c, prompt_plan(c).parts) : -1;
}

// Query rows of the segments (row cu[s] + i at position start[s] + i) over the cache, their own keys
// included; rows in no segment are left as they are.
int amdk8s_llm_kv8_prompt(const void* call, float scale, void* work, long work_floats, void* stream) {
  const AttnCall& c = *static_cast<const AttnCall*>(call);
  if (!good_prompt(c) || !c.out.at || c.x8) return 2;
  const PromptPlan plan = prompt_plan(c);
  const long need = work_floats_of(c, plan.parts);
  if (need > work_floats || (need && (!work || ((uintptr_t)work & 15)))) return 2;
  if (plan.units * c.c.hkv > 0x7fffffffL || plan.parts > 65535 || (plan.parts > 1 && c.n > 65535)) return 2;
  AttnArgs a = make_attn(c, scale, need ? work : nullptr, plan.parts);
  a.units = (int)plan.units;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(plan.units * c.c.hkv), (unsigned)plan.parts);
  return by_format(c.c, [&](auto d, auto f) -> int {
    constexpr int DD = decltype(d)::value;
    constexpr bool F8 = decltype(f)::value;
    auto go = [&](auto rw, auto slots) {
      constexpr int RW = decltype(rw)::value, SL = decltype(slots)::value;
      if (c.type == kF16) hipLaunchKernelGGL((kv8_prompt_kernel<DD, F8, kF16, RW, SL>), grid, dim3(64 * RW * SL), 0, st, a);
      else hipLaunchKernelGGL((kv8_prompt_kernel<DD, F8, kBF16, RW, SL>), grid, dim3(64 * RW * SL), 0, st, a);
    };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    if (plan.slots == 2) go(I4{}, I2{});
    else if (plan.rw == 8) go(I8{}, I1{});
    else go(I4{}, I1{});
    if (need) {
      const dim3 rows((unsigned)c.heads, (unsigned)c.n);
      if (c.type == kF16) hipLaunchKernelGGL((kv8_join_kernel<DD, kF16, 1, false>), rows, dim3(64), 0, st, a);
      else hipLaunchKernelGGL((kv8_join_kernel<DD, kBF16, 1, false>), rows, dim3(64), 0, st, a);
    }
    return launched();
  });
}

}  // extern "C"
