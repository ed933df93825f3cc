// K/V cache held in microscaled 8 or 4 bits: writing it, reading it back and
// attention over it (gfx950, head_dim 64).
//
// Quantisation.  32 consecutive values of a row share a power of two 2^E; an
// element is the nearest e4m3 or e2m1 number to x / 2^E (ties to the even
// code: the rounding of v_cvt_scalef32_pk_{fp8,fp4}_bf16).  E is the smallest
// exponent, -110 at least, for which no element saturates, max|x| <= 448 2^E
// (6 2^E), held as the byte E + 127.  So every stored value is a normal bf16
// number or zero, so reading back and the products below use
// exactly the stored value.  Magnitudes over 1.5 2^127 are stored as that (the
// next e2m1 step would be infinite).  A block that holds an infinity or a NaN
// gets the scale byte 0xff and zero codes and reads as NaN throughout.
//
// Layout.  A record holds 32 tokens of one head of one sequence in the order
// in which the attention's MFMAs take them, so that a wave reads it as whole
// consecutive kilobytes, straight into operand registers:
//   K (A operand of S^T = K . Q^T): lane (g, s & 15), g = lane / 16, holds for
//     token half s >> 4 and depth half ks the codes of d = 32 ks + 8 g + 0..7;
//     4 bits: one dword [half][ks] of the lane's 16 bytes; 8 bits: two dwords
//     at [half] kilobyte, [ks] half of the lane's 16 bytes.
//   V (A operand of O^T = V^T . P^T): lane (g, d & 15) holds, for depth blocks
//     blk = d >> 5 and token halves, the codes of the tokens 16 half + 4 g + 0..3
//     (the order in which S^T's accumulators become the operand P^T), depths d
//     and d + 16 of a token side by side: they share a scale, so one conversion
//     gives both.  4 bits: a dword [blk][half], a byte a token; 8 bits: [blk]
//     kilobyte, two dwords [half] of the lane's 16 bytes, 2 bytes a token.
//   K scales: byte [s & 15][half][ks]; V scales: byte [g][d >> 5][8 tokens].
// 4 bits: 1024 + 1024 + 64 + 64 bytes; 8 bits: 2048 + 2048 + 64 + 64.
//
// Positions.  The first `sinks` positions have records of their own; position
// p >= sinks is token (p - sinks) % 32 of ring tile u = (p - sinks) / 32, held
// in record u % (ring / 32) after the sinks'.  Per sequence the state is the
// number of tokens n and the first ring tile still held, lo; lo = kLost marks
// a sequence whose contents cannot be vouched for (a position that skips
// ahead was written), until it is written from position 0 again.
//
// MI355X, against a large copy's 5.15 TB/s: 4 x 32768 uneven rows of 5 heads
// written at 4 bits 38 us (159 MB, 4.2 TB/s) and read back 30 (201 MB, 6.7: the
// L2s hold part); attention of one token over 16 x 65536 tokens of 4 bits 73 + 4
// (357 MB, 4.9), over 32 contexts of 4096 to 8192 of 8 bits 23 + 4 (130 MB, 5.6);
// 2 x 1000 rows with a window of 2048 28 (15.8 GFLOP, 560 TFLOP/s).
#include "attention_tile.h"

namespace {

constexpr int TOK = 32;                 // tokens of a record
constexpr int kMaxPos = 1 << 30;        // positions stay below it
constexpr int kLost = 0x7fffffff;
constexpr int kCUs = 256;
constexpr int kMaxSplits = 256;
constexpr unsigned kMaxArrivals = 64;

template <int BITS> constexpr int kPart = TOK * D * BITS / 8;      // bytes of K (or V) codes
template <int BITS> constexpr int kRec = 2 * kPart<BITS> + 128;

struct Cache {
  uint8_t* data;
  int* state;                           // [batch][4]: n, lo, arrivals, -
  int heads, sinks, sink_tiles, ring_tiles;
};

__device__ __forceinline__ long record(const Cache& c, int b, int h, int tile) {
  return ((long)b * c.heads + h) * (c.sink_tiles + c.ring_tiles) + tile;
}

// What a write of `count` rows at position p0 does to a sequence.
struct Span {
  int p0, n, lo;                        // first position, tokens and lo afterwards
};
__device__ __forceinline__ Span write_span(const Cache& c, int n, int lo, int p0, int count) {
  Span s;
  s.p0 = p0;
  if (p0 < 0 || p0 > n || p0 > kMaxPos - count || (lo == kLost && p0 != 0)) {
    s.n = n;
    s.lo = kLost;
    return s;
  }
  s.n = p0 + count;
  // nothing of the ring is kept when the write begins inside the sinks
  const int keep = p0 <= c.sinks ? 0 : lo;
  const int last = s.n > c.sinks ? (s.n - 1 - c.sinks) >> 5 : -1;
  s.lo = max(keep, last - c.ring_tiles + 1);
  return s;
}

// The records that hold positions [p0, n): first the sinks', then the ring's
// from tile u0.
struct Tiles {
  int s0, ns, u0, nr;
};
__device__ __forceinline__ Tiles tiles_of(const Cache& c, int p0, int n) {
  Tiles t = {0, 0, 0, 0};
  if (p0 >= n) return t;
  if (p0 < c.sinks) {
    t.s0 = p0 >> 5;
    t.ns = ((min(n, c.sinks) - 1) >> 5) - t.s0 + 1;
  }
  if (n > c.sinks) {
    t.u0 = (max(p0, c.sinks) - c.sinks) >> 5;
    t.nr = ((n - 1 - c.sinks) >> 5) - t.u0 + 1;
  }
  return t;
}

// ------------------------------------------------------------------ write ---
struct AppendArgs {
  Cache c;
  const bf16 *k, *v;
  long ldk, k_bs, ldv, v_bs;
  const int *counts, *at;
  int rows;
};

// Scale byte of a block whose largest magnitude has the bf16 bits `top`.
template <int BITS> __device__ __forceinline__ int scale_byte(unsigned top) {
  if (top >= 0x7f80) return 255;
  top = min(top, 0x7f40u);
  // top = 2^(e-127) (1 + m/128): the largest element is 1.5 2^2 (1.75 2^8)
  const int e = (int)(top >> 7), m = (int)(top & 127);
  const int s = BITS == 4 ? e - 2 + (m > 0x40) : e - 8 + (m > 0x60);
  return max(s, 17);
}

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Codes of 8 values (element i at 4 i or 8 i bits); byte = their scale byte.
template <int BITS> __device__ __forceinline__ u32x2 encode8(u32x4 x, int byte) {
  u32x2 r = {0u, 0u};
  if (byte == 255) return r;
  const float sc = __uint_as_float((unsigned)byte << 23);
  bf16x2 p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned w = x[i];
    if (BITS == 8 && byte == 246) {      // +-1.5 2^127 (e2m1 saturates there itself)
      unsigned a = w & 0x7fff, b = (w >> 16) & 0x7fff;
      a = min(a, 0x7f40u) | (w & 0x8000u);
      b = min(b, 0x7f40u) | ((w >> 16) & 0x8000u);
      w = a | (b << 16);
    }
    p[i] = __builtin_bit_cast(bf16x2, w);
  }
  if constexpr (BITS == 4) {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[0], sc, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[1], sc, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[2], sc, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[3], sc, 3);
    r[0] = w;
  } else {
    s16x2 a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, p[0], sc, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, p[1], sc, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, p[2], sc, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, p[3], sc, true);
    r[0] = __builtin_bit_cast(unsigned, a);
    r[1] = __builtin_bit_cast(unsigned, b);
  }
  return r;
}

// largest magnitude (bf16 bits) of 8 values, and of those of the 4 lanes of a block
__device__ __forceinline__ unsigned top8(u32x4 x) {
  unsigned t = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) t = max(t, max(x[i] & 0x7fff, (x[i] >> 16) & 0x7fff));
  return t;
}
__device__ __forceinline__ unsigned block_top(u32x4 x) {
  unsigned t = top8(x);
  t = max(t, (unsigned)__shfl_xor((int)t, 1));
  return max(t, (unsigned)__shfl_xor((int)t, 2));
}

// One wave builds one record in LDS and stores it whole.  Lane l takes rows
// 8 i + l / 8, i = 0..3, and the 8 values of chunk l % 8: their codes are one
// dword (two) of the K operand; the V operand's are scattered as bytes, put
// together by the lanes of depths d and d + 16 at 4 bits.  A record that keeps older tokens is read first.
//
// The last workgroup of a sequence to have read its state stores the new one;
// with more than kMaxArrivals of them advance_kernel does, since the arrivals at
// one address take 6 ns each (4 x 32768 rows of 5 heads, 1280 workgroups a
// sequence: 72 us against 39 + 4).
template <int BITS>
__global__ __launch_bounds__(1024) void append_kernel(AppendArgs a) {
  constexpr int PART = kPart<BITS>, REC = kRec<BITS>;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int b = blockIdx.y;
  const int n_old = c.state[4 * b], lo_old = c.state[4 * b + 1];
  const int count = a.counts ? min(max(a.counts[b], 0), a.rows) : a.rows;
  const Span sp = write_span(c, n_old, lo_old, a.at ? a.at[b] : n_old, count);
  Tiles t = tiles_of(c, sp.p0, sp.lo == kLost ? sp.p0 : sp.p0 + count);
  {  // of a long write only the tiles that stay
    const int skip = max(0, sp.lo == kLost ? 0 : sp.lo - t.u0);
    if (t.nr > 0) { t.u0 += skip; t.nr -= skip; }
  }
  uint8_t* rec = lds + wave * REC;
  const int units = (t.ns + t.nr) * c.heads;
  for (int base = blockIdx.x * waves; base < units; base += gridDim.x * waves) {
    const int unit = base + wave;
    const bool on = unit < units;
    const int ti = on ? unit / c.heads : 0, h = on ? unit - ti * c.heads : 0;
    const bool sink = ti < t.ns;
    const int u = sink ? t.s0 + ti : t.u0 + ti - t.ns;
    const int pos0 = sink ? u * TOK : c.sinks + u * TOK;
    const int pend = sink ? min(c.sinks, sp.n) : sp.n;
    uint8_t* out = c.data + record(c, b, h, sink ? u : c.sink_tiles + u % c.ring_tiles) * REC;
    u32x4 xk[4], xv[4];
    bool in[4];
    if (on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = pos0 + 8 * i + (lane >> 3);
        in[i] = p >= sp.p0 && p < pend;
        const long r = in[i] ? p - sp.p0 : 0;
        const int col = h * D + (lane & 7) * 8;
        xk[i] = in[i] ? *(const u32x4*)(a.k + b * a.k_bs + r * a.ldk + col) : u32x4{0, 0, 0, 0};
        xv[i] = in[i] ? *(const u32x4*)(a.v + b * a.v_bs + r * a.ldv + col) : u32x4{0, 0, 0, 0};
      }
      const bool keep = pos0 < sp.p0;
      for (int i = lane; i < REC / 16; i += 64)
        ((u32x4*)rec)[i] = keep ? ((const u32x4*)out)[i] : u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    if (on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = 8 * i + (lane >> 3), ch = lane & 7, half = s >> 4, s16 = s & 15;
        const int kb = scale_byte<BITS>(block_top(xk[i])), vb = scale_byte<BITS>(block_top(xv[i]));
        const u32x2 kc = encode8<BITS>(xk[i], kb), vc = encode8<BITS>(xv[i], vb);
        const int ks = ch >> 2, kl = (ch & 3) * 16 + s16;
        const int g = s16 >> 2, j = half * 4 + (s & 3);
        if constexpr (BITS == 4) {
          if (in[i]) *(unsigned*)(rec + kl * 16 + (half * 2 + ks) * 4) = kc[0];
          // depths d and d + 16 share a byte: the lanes of either (ch, ch ^ 2)
          // store half of the 8 bytes
          const unsigned oc = __shfl_xor(vc[0], 2);
          const bool up = ch & 2;
          const unsigned lo4 = up ? oc : vc[0], hi4 = up ? vc[0] : oc;
          if (in[i]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d8 = (up ? 4 : 0) + e;
              rec[PART + (g * 16 + (ch & 1) * 8 + d8) * 16 + (ks * 2 + half) * 4 + (s & 3)] =
                  (uint8_t)(((lo4 >> (4 * d8)) & 15u) | (((hi4 >> (4 * d8)) & 15u) << 4));
            }
          }
        } else if (in[i]) {
          *(u32x2*)(rec + half * 1024 + kl * 16 + ks * 8) = kc;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            rec[PART + ks * 1024 + (g * 16 + (ch & 1) * 8 + e) * 16 + half * 8 + (s & 3) * 2 + ((ch >> 1) & 1)] =
                (uint8_t)(vc[e >> 2] >> (8 * (e & 3)));
        }
        if (in[i] && (ch & 3) == 0) {
          rec[2 * PART + s16 * 4 + half * 2 + ks] = (uint8_t)kb;
          rec[2 * PART + 64 + g * 16 + ks * 8 + j] = (uint8_t)vb;
        }
      }
    }
    __syncthreads();
    if (on)
      for (int i = lane; i < REC / 16; i += 64) ((u32x4*)out)[i] = ((const u32x4*)rec)[i];
    __syncthreads();
  }
  __syncthreads();                      // every wave has read the old state
  if (threadIdx.x == 0 && gridDim.x <= kMaxArrivals && __hip_atomic_fetch_add(&c.state[4 * b + 2], 1, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1) {
    c.state[4 * b] = sp.n;
    c.state[4 * b + 1] = sp.lo;
    c.state[4 * b + 2] = 0;
  }
}

__global__ void advance_kernel(AppendArgs a, int batch) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int n = a.c.state[4 * b];
  const int count = a.counts ? min(max(a.counts[b], 0), a.rows) : a.rows;
  const Span s = write_span(a.c, n, a.c.state[4 * b + 1], a.at ? a.at[b] : n, count);
  a.c.state[4 * b] = s.n;
  a.c.state[4 * b + 1] = s.lo;
}

__global__ void reset_kernel(int* state, int batch) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < 4 * batch) state[i] = 0;
}

// --------------------------------------------------------------- decoding ---
// The scale operand of v_cvt_scalef32_* counts by its exponent field alone, so
// byte i of a dword becomes a scale by one shift.
template <int I> __device__ __forceinline__ float scale_of(unsigned w) {
  return __uint_as_float(I == 3 ? w >> 1 : w << (23 - 8 * I));
}

template <int BITS, int PAIR>             // codes 2 PAIR, 2 PAIR + 1 of 8
__device__ __forceinline__ unsigned decode2(u32x2 w, float sc) {
  if constexpr (BITS == 4)
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, PAIR));
  else
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[PAIR >> 1], sc, PAIR & 1));
}

// 8 codes of one scale
template <int BITS> __device__ __forceinline__ bf16x8 decode8(u32x2 w, float sc) {
  const u32x4 r = {decode2<BITS, 0>(w, sc), decode2<BITS, 1>(w, sc), decode2<BITS, 2>(w, sc),
                   decode2<BITS, 3>(w, sc)};
  return __builtin_bit_cast(bf16x8, r);
}

// A record in a wave's registers.
template <int BITS> struct Rec {
  u32x4 k[BITS / 4], v[BITS / 4];
  unsigned ks;                          // scales of token (lane & 15): [half][ks]
  u32x4 vs;                             // scales of the lane's 8 tokens: [d >> 5][8]
  __device__ __forceinline__ void load(const uint8_t* p, int lane) {
    constexpr int PART = kPart<BITS>;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
      k[i] = *(const u32x4*)(p + i * 1024 + lane * 16);
      v[i] = *(const u32x4*)(p + PART + i * 1024 + lane * 16);
    }
    ks = *(const unsigned*)(p + 2 * PART + (lane & 15) * 4);
    vs = *(const u32x4*)(p + 2 * PART + 64 + (lane >> 4) * 16);
  }
  __device__ __forceinline__ u32x2 kw(int half, int s) const {
    return BITS == 4 ? u32x2{k[0][half * 2 + s], 0u}
                     : u32x2{k[BITS == 4 ? 0 : half][s * 2], k[BITS == 4 ? 0 : half][s * 2 + 1]};
  }
  __device__ __forceinline__ void store(uint8_t* p, int lane) const {
    constexpr int PART = kPart<BITS>;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
      *(u32x4*)(p + i * 1024 + lane * 16) = k[i];
      *(u32x4*)(p + PART + i * 1024 + lane * 16) = v[i];
    }
    if (lane < 16) *(unsigned*)(p + 2 * PART + lane * 4) = ks;
    if ((lane & 15) == 0) *(u32x4*)(p + 2 * PART + 64 + (lane >> 4) * 16) = vs;
  }
  // Token `slot` (the same in every lane) becomes the row kn, vn; the first
  // token of a record clears it.
  __device__ __forceinline__ void insert(const bf16* kn, const bf16* vn, int slot, int lane) {
    const int grp = lane >> 4, col = lane & 15, half = slot >> 4, s16 = slot & 15;
    if (slot == 0) {
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) k[i] = v[i] = u32x4{0, 0, 0, 0};
      ks = 0;
      vs = u32x4{0, 0, 0, 0};
    }
    auto put = [](unsigned& w, unsigned x, int shift, unsigned width) {
      const unsigned m = width << shift;
      w = (w & ~m) | ((x << shift) & m);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const u32x4 x = *(const u32x4*)(kn + s * 32 + grp * 8);
      unsigned top = top8(x);
      top = max(top, (unsigned)__shfl_xor((int)top, 16));
      top = max(top, (unsigned)__shfl_xor((int)top, 32));
      const int byte = scale_byte<BITS>(top);
      const u32x2 code = encode8<BITS>(x, byte);
      if (col == s16) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (hf == half) {
            if constexpr (BITS == 4) {
              k[0][hf * 2 + s] = code[0];
            } else {
              k[hf][s * 2] = code[0];
              k[hf][s * 2 + 1] = code[1];
            }
          }
        put(ks, byte, 8 * (half * 2 + s), 255u);
      }
    }
    const unsigned short* vb = reinterpret_cast<const unsigned short*>(vn);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const u32x4 x = {(unsigned)vb[blk * 32 + col] | (unsigned)vb[blk * 32 + 16 + col] << 16, 0u, 0u, 0u};
      unsigned top = top8(x);
#pragma unroll
      for (int m = 1; m < 16; m <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, m));
      const int byte = scale_byte<BITS>(top);
      const u32x2 code = encode8<BITS>(x, byte);
      if (grp == (s16 >> 2)) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (q == half) {
            if constexpr (BITS == 4) {
              unsigned y = v[0][blk * 2 + q];
              put(y, code[0], 8 * (slot & 3), 255u);
              v[0][blk * 2 + q] = y;
            } else {
#pragma unroll
              for (int w = 0; w < 2; ++w)
                if (w == ((slot >> 1) & 1)) {
                  unsigned y = v[blk][q * 2 + w];
                  put(y, code[0], 16 * (slot & 1), 0xffffu);
                  v[blk][q * 2 + w] = y;
                }
            }
            unsigned y = vs[blk * 2 + q];
            put(y, byte, 8 * (slot & 3), 255u);
            vs[blk * 2 + q] = y;
          }
      }
    }
  }
  template <int HALF, int S> __device__ __forceinline__ bf16x8 kfrag() const {
    return decode8<BITS>(kw(HALF, S), scale_of<HALF * 2 + S>(ks));
  }
  // the operands of depths 32 blk + 0..15 and + 16..31: a conversion per token,
  // then the halves of two tokens are sorted out
  template <int BLK> __device__ __forceinline__ void vfrags(bf16x8& lo, bf16x8& hi) const {
    unsigned t[8];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const u32x2 w = BITS == 4 ? u32x2{v[0][BLK * 2 + hf], 0u}
                                : u32x2{v[BITS == 4 ? 0 : BLK][hf * 2], v[BITS == 4 ? 0 : BLK][hf * 2 + 1]};
      const unsigned sc = vs[BLK * 2 + hf];
      t[hf * 4 + 0] = decode2<BITS, 0>(w, scale_of<0>(sc));
      t[hf * 4 + 1] = decode2<BITS, 1>(w, scale_of<1>(sc));
      t[hf * 4 + 2] = decode2<BITS, 2>(w, scale_of<2>(sc));
      t[hf * 4 + 3] = decode2<BITS, 3>(w, scale_of<3>(sc));
    }
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100u);
      b[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302u);
    }
    lo = __builtin_bit_cast(bf16x8, a);
    hi = __builtin_bit_cast(bf16x8, b);
  }
};

// ------------------------------------------------------------------- read ---
struct ReadArgs {
  Cache c;
  bf16 *k, *v;
  long ldk, k_bs, ldv, v_bs;
  const int* starts;
  int start, rows;
};

// One wave decodes one record; K leaves as the operand's own 8 values a lane,
// V through LDS.  Rows that the cache does not hold (behind the last token,
// fallen out of the ring, of a lost sequence) are zeros.
template <int BITS>
__global__ __launch_bounds__(64) void read_kernel(ReadArgs a) {
  constexpr int LD = D + 8;
  __shared__ __attribute__((aligned(16))) bf16 sv[TOK * LD];
  const Cache& c = a.c;
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int grp = lane >> 4, col = lane & 15;
  const int n = c.state[4 * b], lo = c.state[4 * b + 1];
  // (positions past kMaxPos do not exist; a start out of range reads zeros)
  const int first = min(max(a.starts ? a.starts[b] : a.start, -kMaxPos), kMaxPos - 1);
  const int p0 = max(first, 0), p1 = first + a.rows;
  const Tiles t = tiles_of(c, p0, p1);
  bf16* ko = a.k + b * a.k_bs + h * D;
  bf16* vo = a.v + b * a.v_bs + h * D;
  const bf16x8 zero = {};
  if (blockIdx.x == 0 && first < 0)
    for (long i = lane; i < 8L * min(a.rows, -first); i += 64) {
      st8(ko + (i >> 3) * a.ldk + (i & 7) * 8, zero);
      st8(vo + (i >> 3) * a.ldv + (i & 7) * 8, zero);
    }
  for (int ti = blockIdx.x; ti < t.ns + t.nr; ti += gridDim.x) {
    const bool sink = ti < t.ns;
    const int u = sink ? t.s0 + ti : t.u0 + ti - t.ns;
    const int pos0 = sink ? u * TOK : c.sinks + u * TOK;
    const int pend = min(p1, sink ? c.sinks : p1);         // rows of this record to write
    const bool held = lo != kLost && (sink || u >= lo) && pos0 < n;
    Rec<BITS> r = {};
    if (held) r.load(c.data + record(c, b, h, sink ? u : c.sink_tiles + u % c.ring_tiles) * kRec<BITS>, lane);
    auto put_k = [&](int half, int s, bf16x8 x) {
      const int p = pos0 + half * 16 + col;
      if (p >= p0 && p < pend)
        st8(ko + (long)(p - first) * a.ldk + s * 32 + grp * 8, held && p < n ? x : zero);
    };
    put_k(0, 0, r.template kfrag<0, 0>());
    put_k(0, 1, r.template kfrag<0, 1>());
    put_k(1, 0, r.template kfrag<1, 0>());
    put_k(1, 1, r.template kfrag<1, 1>());
    bf16x8 vf[4];
    r.template vfrags<0>(vf[0], vf[1]);
    r.template vfrags<1>(vf[2], vf[3]);
#pragma unroll
    for (int td = 0; td < 4; ++td)
#pragma unroll
      for (int j = 0; j < 8; ++j) sv[((j >> 2) * 16 + 4 * grp + (j & 3)) * LD + td * 16 + col] = vf[td][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = 8 * i + (lane >> 3), p = pos0 + s;
      if (p >= p0 && p < pend)
        st8(vo + (long)(p - first) * a.ldv + (lane & 7) * 8,
            held && p < n ? *(const bf16x8*)(sv + s * LD + (lane & 7) * 8) : zero);
    }
    __syncthreads();
  }
}

// -------------------------------------------------------------- attention ---
struct AttendArgs {
  Cache c;
  const bf16* q;
  long ldq, q_bs;
  bf16* o;
  long ldo, o_bs;
  const int* counts;
  int rows, group, window;
  unsigned group_inv;         // j / group = (j * group_inv) >> 32 for the columns j
  float scale_log2;
  int splits;
  float *part, *stat;         // [batch * heads][columns][splits] x 64 and x 2
  // one new row per sequence to be written on the way (NULL: none)
  const bf16 *k, *v;
  long k_bs, v_bs;
  const int* at;
};

// What a call sees of one sequence.
struct View {
  int first, count;           // position of query row 0, rows
  bool lost;                  // a position that the call needs is gone
};
__device__ __forceinline__ View view_of(const AttendArgs& a, int b, int n, int lo) {
  View v;
  v.count = a.counts ? min(max(a.counts[b], 0), a.rows) : a.rows;
  v.first = n - v.count;
  const int need = max(a.c.sinks, a.window ? v.first - a.window + 1 : 0);
  v.lost = lo == kLost || v.first < 0 || (need < n && (need - a.c.sinks) >> 5 < lo);
  return v;
}

__device__ __forceinline__ int row_of(const AttendArgs& a, int j) {
  return a.group_inv ? (int)__umulhi((unsigned)j, a.group_inv) : j;
}

// Output of one column: 4 depths from d on; rows behind the count are zeros.
__device__ __forceinline__ void put_out(bf16* out, f32x4 o, float l, const View& v, int r) {
  const float inv = l > 0.f ? 1.0f / l : l;        // nothing visible: 0; NaN stays
  bf16x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = f2bf(r >= v.count ? 0.f : v.lost ? __builtin_nanf("") : o[i] * inv);
  *reinterpret_cast<bf16x4*>(out) = y;
}

// Columns: column j of a KV head is query row j / group of query head
// j % group of the head's group, so all the query heads that share a KV head
// share each record that a wave decodes.  A workgroup holds QT tiles of 16
// columns; its 4 waves take turns at the records and are joined through LDS.
// The records of a call are split over blockIdx.y too when there are few
// columns; the parts (reference, sum, unscaled output) are then joined by
// join_kernel.
//
// S^T[token, column] = K . Q^T and O^T[d, column] = V^T . P^T, so a lane owns
// one column (lane & 15); the accumulators of S^T are the operand P^T as they
// stand.  The sum of the rounded probabilities is an MFMA with a row of ones.
//
// Softmax needs no maximum where exp(s) itself neither over- nor underflows: any
// reference gives the same quotient, and bf16 keeps fp32's range.  So the first
// time over the records takes the reference 0.  A wave of which a column's sum
// leaves [2^-40, 2^100], or an output 2^100 (also by infinities and NaNs, even
// from behind the mask, as 0 * NaN), goes over its records once more, following
// the maximum, and a column then meets only what it sees, NaN blocks apart.
//
// Up to 64 columns a KV head (QT < 4) the probabilities go into the products as
// bf16 and a bf16 remainder: what they would be off by, 2^-9 in the mean square,
// is as much as the output's own rounding.  Such calls read or wait, so it costs
// little there (16 x 65536 tokens 70 -> 74 us, 8 bits nothing); with more columns
// the products are what costs, and the probabilities are rounded once, as in
// attention_kernel.
//
// What bounds it: one row reads its records at a copy's rate once they are
// enough to fill the chip; many rows are bound by issue, a record and 64 columns
// being 36 MFMAs (576 cycles) and ~170 vector instructions (~850 with the 32
// exponentials), 1370 cycles measured at two waves per SIMD.  Short calls are
// launch (2 us), the loads of state, then Q and records (1.5), and the joins.
//
// PF records are in registers or on their way to them.
template <int BITS, int QT> constexpr int kAhead = QT == 1 ? (BITS == 4 ? 3 : 2) : 8 / BITS;

// NEW: one new row per sequence is written on the way.
template <int BITS, int QT, bool NEW>
__global__ __launch_bounds__(256, QT == 4 ? 2 : 3) void attend_kernel(AttendArgs a) {
  constexpr int PF = kAhead<BITS, QT>, KW = 4, LD = D + 4;
  constexpr bool TWO = QT < 4;                     // probabilities in two bf16 terms
  // per wave and column: 64 depths, reference, sum
  __shared__ __attribute__((aligned(16))) float s_part[KW][16 * QT][LD];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = lane >> 4, col = lane & 15;
  const int b = blockIdx.z / c.heads, h = blockIdx.z - b * c.heads;
  const int ncol = a.rows * a.group;
  const int col0 = blockIdx.x * QT * 16;
  Span span = {0, c.state[4 * b], c.state[4 * b + 1]};
  if constexpr (NEW) {
    const int add = a.counts ? min(max(a.counts[b], 0), 1) : 1;
    span = write_span(c, span.n, span.lo, a.at ? a.at[b] : span.n, add);
  }
  const View view = view_of(a, b, span.n, span.lo);
  const int first = view.first, count = view.count;

  int qpos[QT];                                    // of this lane's column; -1: none
  bf16x8 qf[QT][2];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int j = min(col0 + t * 16 + col, ncol - 1);
    const int r = row_of(a, j), hh = h * a.group + j - r * a.group;
    qpos[t] = r < count ? first + r : -1;
    const bf16* q = a.q + b * a.q_bs + r * a.ldq + hh * D;
#pragma unroll
    for (int s = 0; s < 2; ++s) qf[t][s] = ld8(q + s * 32 + grp * 8);
  }
  // positions of the workgroup's first and last row
  const int r0 = row_of(a, col0), r1 = row_of(a, min(col0 + QT * 16, ncol) - 1);
  const int qlo = first + min(r0, count - 1), qhi = first + min(r1, count - 1);

  f32x4 o[QT][5];
  float m_run[QT], m_off[QT];
  const float cs = a.scale_log2;
  auto clear = [&](float m) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
      for (int i = 0; i < 5; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[t] = m;
      m_off[t] = 0.f;
    }
  };
  clear(-INFINITY);
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = f2bf(1.0f);

  if (r0 < count && !view.lost) {
    const int wlo = a.window ? max(0, qlo - a.window + 1) : 0;
    // records: the sinks that some column sees, then the ring from `wlo`
    const int ns = (min(c.sinks, qhi + 1) + TOK - 1) / TOK;
    const int u0 = max(wlo - c.sinks, 0) >> 5;
    const int nr = qhi >= c.sinks ? max(((qhi - c.sinks) >> 5) - u0 + 1, 0) : 0;
    const int total = ns + nr;
    const int per = max((total + a.splits - 1) / a.splits, min(KW * 4, total));
    const int t0 = blockIdx.y * per, t1 = min(total, t0 + per);
    const int from = t0 + kw;
    const uint8_t* base = c.data + record(c, b, h, 0) * kRec<BITS>;
    // record of place ti in the list (past the end: the last one)
    const int at_u = u0 % c.ring_tiles;
    auto addr = [&](int ti) {
      ti = min(ti, t1 - 1);
      int u = ti;
      if (ti >= ns) {
        u = at_u + ti - ns;                        // < 2 ring_tiles: nr <= ring_tiles
        u = c.sink_tiles + (u >= c.ring_tiles ? u - c.ring_tiles : u);
      }
      return base + (long)u * kRec<BITS>;
    };
    // One record.  FOLLOW: the second time over them, see above.
    auto step = [&](auto FOLLOW, Rec<BITS>& r, int ti) __attribute__((always_inline)) {
      const bool sink = ti < ns;
      const int pos0 = sink ? ti * TOK : c.sinks + (u0 + ti - ns) * TOK;
      const int plim = sink ? c.sinks : kMaxPos;    // (positions of the ring are no sinks)
      // all 32 positions are visible to every column of the workgroup
      const bool full = pos0 + TOK - 1 <= qlo && pos0 + TOK <= plim &&
                        (!a.window || pos0 > qhi - a.window || pos0 + TOK <= c.sinks);
      // (a wave at its matrix products goes before one at its exponentials:
      // 2 x 1000 rows 35.8 -> 34.7 us, 16 x 65536 tokens 79 -> 76)
      __builtin_amdgcn_s_setprio(1);
      f32x4 sc[QT][2];
      {
        const bf16x8 k00 = r.template kfrag<0, 0>(), k01 = r.template kfrag<0, 1>();
        const bf16x8 k10 = r.template kfrag<1, 0>(), k11 = r.template kfrag<1, 1>();
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
          x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k00, qf[t][0], x, 0, 0, 0);
          y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k10, qf[t][0], y, 0, 0, 0);
          sc[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k01, qf[t][1], x, 0, 0, 0);
          sc[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k11, qf[t][1], y, 0, 0, 0);
        }
      }
      auto sees = [&](int t, int i) {               // token (i >> 2) * 16 + 4 grp + (i & 3)
        const int before = !sink && a.window ? qpos[t] - a.window : -1;
        const int n = min(qpos[t], plim - 1) - before;          // (before, before + n]
        return (unsigned)(pos0 + grp * 4 - before - 1 + (i >> 2) * 16 + (i & 3)) < (unsigned)n;
      };
      if (!full) {
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sc[t][i >> 2][i & 3] = sees(t, i) ? sc[t][i >> 2][i & 3] : -INFINITY;
      }
      if constexpr (decltype(FOLLOW)::value) {
        // the maximum moves when a score passes it by 2^8 (exp2 units)
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float mx = sc[t][0][0];
#pragma unroll
          for (int i = 1; i < 8; ++i) mx = smax(mx, sc[t][i >> 2][i & 3]);
          mx = max_xor32(max_xor16(mx));
          const bool grow = mx * cs > m_run[t] * cs + 8.f;
          if (__builtin_amdgcn_ballot_w64(grow)) {
            const float m_new = smax(m_run[t], mx);
            const float alpha = m_run[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[t] - m_new) * cs);
#pragma unroll
            for (int i = 0; i < 5; ++i) o[t][i] *= alpha;
            m_run[t] = m_new;
            m_off[t] = m_new == -INFINITY ? 0.f : -m_new * cs;
          }
        }
        // NaN blocks (scale byte 0xff) count as 0 in V and are added to the
        // columns that see them
#pragma unroll 1
        for (int blk = 0; blk < 2; ++blk) {
          const unsigned v0 = blk ? r.vs[2] : r.vs[0], v1 = blk ? r.vs[3] : r.vs[1];
          unsigned nan_bits = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            nan_bits |= ((((j < 4 ? v0 : v1) >> (8 * (j & 3))) & 255u) == 255u ? 1u : 0u) << j;
          if (!__builtin_amdgcn_ballot_w64(nan_bits != 0)) continue;
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            bf16x8 pn;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              pn[j] = f2bf(((nan_bits >> j) & 1u) && sees(t, j) ? __builtin_nanf("") : 0.f);
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pn, z, 0, 0, 0);
#pragma unroll
            for (int td = 0; td < 4; ++td)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][td][i] += (td >> 1) == blk ? z[i] : 0.f;
          }
          unsigned w0 = 0, w1 = 0;               // bytes 0xff: any valid scale
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w0 |= ((nan_bits >> j) & 1u ? 0x80u : 0u) << (8 * j);
            w1 |= ((nan_bits >> (4 + j)) & 1u ? 0x80u : 0u) << (8 * j);
          }
          r.vs[0] ^= blk ? 0u : w0;
          r.vs[1] ^= blk ? 0u : w1;
          r.vs[2] ^= blk ? w0 : 0u;
          r.vs[3] ^= blk ? w1 : 0u;
        }
      }
      __builtin_amdgcn_s_setprio(0);
      bf16x8 pf[QT], pl[TWO ? QT : 1];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i >> 2][i & 3], cs, m_off[t]));
          pf[t][i] = f2bf(e);
          if constexpr (TWO) pl[t][i] = f2bf(e - bf2f(pf[t][i]));
        }
        o[t][4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[t], o[t][4], 0, 0, 0);
        if constexpr (TWO) o[t][4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pl[t], o[t][4], 0, 0, 0);
      }
      __builtin_amdgcn_s_setprio(1);
      bf16x8 va, vb;
      auto product = [&](int td, bf16x8 vf) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          o[t][td] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t], o[t][td], 0, 0, 0);
          if constexpr (TWO) o[t][td] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[t], o[t][td], 0, 0, 0);
        }
      };
      r.template vfrags<0>(va, vb);
      product(0, va);
      product(1, vb);
      r.template vfrags<1>(va, vb);
      product(2, va);
      product(3, vb);
    };
    // the newest record, where the new row goes: its wave takes it first
    const bool newest = NEW && t1 == total && kw == ((total - 1 - t0) & (KW - 1));
    const int mine = from < t1 ? (t1 - 1 - from) / KW + 1 : 0;       // records of this wave
    auto place = [&](int i) {                                        // its i-th one
      return NEW && newest ? (i == 0 ? total - 1 : from + (i - 1) * KW) : from + i * KW;
    };
    auto insert = [&](Rec<BITS>& r) {
      const int slot = (span.p0 < c.sinks ? span.p0 : span.p0 - c.sinks) & (TOK - 1);
      r.insert(a.k + b * a.k_bs + h * D, a.v + b * a.v_bs + h * D, slot, lane);
    };
    if (mine > 0) {
      Rec<BITS> r[PF];
#pragma unroll
      for (int i = 0; i < PF; ++i) r[i].load(addr(place(i)), lane);
      if (NEW && newest) {
        insert(r[0]);
        r[0].store(const_cast<uint8_t*>(addr(total - 1)), lane);
      }
      for (int at = 0; at < mine; at += PF) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
          if (at + i >= mine) break;
          step(std::false_type{}, r[i], place(at + i));
          r[i].load(addr(place(at + i + PF)), lane);
        }
      }
      bool bad = false;
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float top = o[t][4][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = smax(top, fabsf(o[t][i][e]));
        bad |= qpos[t] >= 0 && !(top < 0x1p100f && o[t][4][0] >= 0x1p-40f);
        m_run[t] = 0.f;
      }
      if (__builtin_amdgcn_ballot_w64(bad)) {
        clear(-INFINITY);
#pragma unroll 1
        for (int at = 0; at < mine; ++at) {
          Rec<BITS> x;
          x.load(addr(place(at)), lane);
          if (NEW && newest && at == 0) insert(x);
          step(std::true_type{}, x, place(at));
        }
      }
    }
  }

  // join the waves: the 4 QT tiles (16 columns x 16 depths) are shared out
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float* part = s_part[kw][t * 16 + col];
#pragma unroll
    for (int td = 0; td < 4; ++td) *(f32x4*)(part + td * 16 + grp * 4) = o[t][td];
    if (grp == 0) {
      part[D] = m_run[t];
      part[D + 1] = o[t][4][0];
    }
  }
  __syncthreads();
  // the last workgroup of a sequence to have read its state moves it on
  if (NEW && threadIdx.x == 64) {
    const int all = gridDim.y * c.heads;
    if (__hip_atomic_fetch_add(&c.state[4 * b + 2], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1) {
      c.state[4 * b] = span.n;
      c.state[4 * b + 1] = span.lo;
      c.state[4 * b + 2] = 0;
    }
  }
  const int jj = (QT == 1 ? 0 : QT == 2 ? kw >> 1 : kw) * 16 + col, j = col0 + jj;
  float mw[KW], m = -INFINITY;
#pragma unroll
  for (int w = 0; w < KW; ++w) {
    mw[w] = s_part[w][jj][D];
    m = smax(m, mw[w]);
  }
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < KW; ++w) {
    mw[w] = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw[w] - m) * cs);
    l += mw[w] * s_part[w][jj][D + 1];
  }
  if (j >= ncol) return;
  const int r = row_of(a, j), hh = h * a.group + j - r * a.group;
  const long at = ((long)blockIdx.z * ncol + j) * a.splits + blockIdx.y;
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int d = ((kw * QT + i) & 3) * 16 + grp * 4;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KW; ++w) y += mw[w] * *(const f32x4*)(s_part[w][jj] + d);
    if (a.splits > 1) *(f32x4*)(a.part + at * D + d) = y;
    else put_out(a.o + b * a.o_bs + r * a.ldo + hh * D + d, y, l, view, r);
  }
  if (a.splits > 1 && grp == 0 && (QT != 1 || kw == 0) && (QT != 2 || !(kw & 1))) {
    a.stat[2 * at] = m;
    a.stat[2 * at + 1] = l;
  }
}

// Joins the parts of the splits: a workgroup per column, its 16 groups of 16
// lanes (4 depths a lane) take turns at the parts.
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a) {
  __shared__ float s_w[kMaxSplits];
  __shared__ f32x4 s_o[4][16];
  const Cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ncol = a.rows * a.group;
  const int j = blockIdx.x;
  const int b = blockIdx.y / c.heads, h = blockIdx.y - b * c.heads;
  const long at = ((long)blockIdx.y * ncol + j) * a.splits;
  // (loads that nothing here decides first: the sequence's state, a lane's part)
  const View view = view_of(a, b, c.state[4 * b], c.state[4 * b + 1]);
  const int d4 = (tid & 15) * 4, s0 = tid >> 4;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (s0 < a.splits) o = *(const f32x4*)(a.part + (at + s0) * D + d4);
  // every wave: the weights of the parts and the sum
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) m = smax(m, a.stat[2 * (at + s)]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) m = smax(m, __shfl_xor(m, x));
  float l = 0.f;
  for (int s = lane; s < a.splits; s += 64) {
    const float ms = a.stat[2 * (at + s)];
    const float w = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ms - m) * a.scale_log2);
    l += w * a.stat[2 * (at + s) + 1];
    if (wave == 0) s_w[s] = w;
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
  __syncthreads();
  o *= s0 < a.splits ? s_w[s0] : 0.f;
#pragma unroll 4
  for (int s = s0 + 16; s < a.splits; s += 16) o += s_w[s] * *(const f32x4*)(a.part + (at + s) * D + d4);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = xor32_sum(xor16_sum(o[i]));
  if (lane < 16) s_o[wave][lane] = o;
  __syncthreads();
  if (tid >= 16) return;
  o = s_o[0][tid] + s_o[1][tid] + s_o[2][tid] + s_o[3][tid];
  const int r = row_of(a, j), hh = h * a.group + j - r * a.group;
  put_out(a.o + b * a.o_bs + r * a.ldo + hh * D + d4, o, l, view, r);
}

bool cache_ok(const svla_kv_cache* c) {
  return c && c->data && c->state && svla_aligned16(c->data) && c->batch > 0 && c->n_kv_heads > 0 &&
         c->head_dim == D && (c->format == SVLA_KV_MXFP4 || c->format == SVLA_KV_MXFP8) &&
         c->sinks >= 0 && c->sinks <= kMaxPos / 2 && c->ring >= TOK && c->ring % TOK == 0 &&
         c->ring <= kMaxPos && c->batch <= 65535 / c->n_kv_heads;
}

Cache device_cache(const svla_kv_cache* c) {
  Cache d;
  d.data = static_cast<uint8_t*>(c->data);
  d.state = c->state;
  d.heads = c->n_kv_heads;
  d.sinks = c->sinks;
  d.sink_tiles = (c->sinks + TOK - 1) / TOK;
  d.ring_tiles = c->ring / TOK;
  return d;
}

bool rows_ok(const void* p, int ld, long bs, int heads) {
  return p && svla_aligned16(p) && ld % 8 == 0 && bs % 8 == 0 && ld >= heads * D;
}

struct Plan {
  int qt, splits;
  dim3 grid;
};

// QT by columns: 64 columns share the decoding of a record (2 x 1000 rows of 3
// heads a KV head: 31.5 us against 34.2 with 32, 53 with 16; 32 x 50 rows over
// 1024 tokens 17.1, 19.0, 33), as long as there are more than that.
//
// Splits: one round of three workgroups a CU, two of 64 columns (16 x 65536
// tokens, one row: 79 us with 720 workgroups, 109 with 240, 80 with 960; one
// sequence of 100003: 14.8 us with 154, 15.8 with 196, whose parts cost the join
// more), each with at least 16 records, 4 a wave, which are on their way at once.
Plan plan_attend(const svla_kv_cache* c, int rows, int hq, int window) {
  Plan p;
  const long ncol = (long)rows * (hq / c->n_kv_heads);
  const long bh = (long)c->batch * c->n_kv_heads;
  p.qt = ncol <= 16 ? 1 : ncol <= 64 ? 2 : 4;
  const long x = (ncol + 16 * p.qt - 1) / (16 * p.qt);
  // records of a sequence, at most
  const long ring = window ? min((long)c->ring, (long)window + rows + 2 * TOK) : (long)c->ring;
  const long tiles = ring / TOK + (c->sinks + TOK - 1) / TOK;
  const long room = kCUs * (p.qt == 4 ? 2 : 3);
  p.splits = (int)max(1L, min(min(room / (x * bh), (tiles + 15) / 16), (long)kMaxSplits));
  p.grid = dim3((unsigned)x, (unsigned)p.splits, (unsigned)bh);
  return p;
}

long scratch_of(const svla_kv_cache* c, const Plan& p, int rows, int hq) {
  return p.splits > 1 ? (long)c->batch * hq * rows * p.splits * (D + 2) * 4 : 0;
}

template <int BITS>
void launch_attend(const Plan& p, const AttendArgs& a, hipStream_t s) {
  if (a.k) {
    if (p.qt == 1) hipLaunchKernelGGL((attend_kernel<BITS, 1, true>), p.grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attend_kernel<BITS, 2, true>), p.grid, dim3(256), 0, s, a);   // (one workgroup's columns: at most 32)
  } else {
    if (p.qt == 1) hipLaunchKernelGGL((attend_kernel<BITS, 1, false>), p.grid, dim3(256), 0, s, a);
    else if (p.qt == 2) hipLaunchKernelGGL((attend_kernel<BITS, 2, false>), p.grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attend_kernel<BITS, 4, false>), p.grid, dim3(256), 0, s, a);
  }
}

// Checks a call's arguments and lays out its plan; rows == 0: no more than that.
int attend_args(const svla_kv_cache* c, const void* q, int ldq, long q_bs, void* o, int ldo,
                long o_bs, int rows, const int* counts, int hq, float scale, int window,
                void* scratch, long scratch_bytes, Plan* p, AttendArgs* a) {
  if (!cache_ok(c) || rows < 0 || hq <= 0 || hq % c->n_kv_heads || window < 0 ||
      !(scale > 0.f) || !(scale < 1e30f))
    return SVLA_EINVAL;
  if (rows == 0) return SVLA_OK;
  if ((long)rows * hq > (1L << 24) || hq / c->n_kv_heads > 255) return SVLA_EINVAL;
  if (!rows_ok(q, ldq, q_bs, hq) || !o || ((uintptr_t)o & 7) || ldo % 4 || o_bs % 4 || ldo < hq * D)
    return SVLA_EINVAL;
  *p = plan_attend(c, rows, hq, window);
  if (scratch_of(c, *p, rows, hq) > scratch_bytes ||
      (p->splits > 1 && (!scratch || !svla_aligned16(scratch))))
    return SVLA_EINVAL;
  *a = AttendArgs{};
  a->c = device_cache(c);
  a->q = static_cast<const bf16*>(q); a->ldq = ldq; a->q_bs = q_bs;
  a->o = static_cast<bf16*>(o); a->ldo = ldo; a->o_bs = o_bs;
  a->counts = counts;
  a->rows = rows;
  a->group = hq / c->n_kv_heads;
  // ceil(2^32 / group): exact while j * group < 2^32 (group 1: no division)
  a->group_inv = a->group == 1 ? 0u : (unsigned)(((1ULL << 32) + a->group - 1) / a->group);
  a->window = min(window, kMaxPos);
  a->scale_log2 = scale * 1.4426950408889634f;
  a->splits = p->splits;
  a->part = static_cast<float*>(scratch);
  a->stat = a->part + (long)c->batch * hq * rows * p->splits * D;
  return SVLA_OK;
}

int run_attend(const svla_kv_cache* c, const Plan& p, const AttendArgs& a, hipStream_t s) {
  if (c->format == SVLA_KV_MXFP4) launch_attend<4>(p, a, s);
  else launch_attend<8>(p, a, s);
  SVLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL(join_kernel, dim3(a.rows * a.group, p.grid.z), dim3(256), 0, s, a);
    SVLA_CHECK_LAUNCH();
  }
  return SVLA_OK;
}

}  // namespace

extern "C" {

long svla_kv_cache_bytes(int batch, int n_kv_heads, int head_dim, int format, int sinks, int ring) {
  svla_kv_cache c = {(void*)16, (int*)16, batch, n_kv_heads, head_dim, format, sinks, ring};
  if (!cache_ok(&c)) return 0;
  const long rec = format == SVLA_KV_MXFP4 ? kRec<4> : kRec<8>;
  return (long)batch * n_kv_heads * ((sinks + TOK - 1) / TOK + ring / TOK) * rec;
}

int svla_kv_reset(const svla_kv_cache* c, svla_stream_t stream) {
  if (!cache_ok(c)) return SVLA_EINVAL;
  hipLaunchKernelGGL(reset_kernel, dim3((4 * c->batch + 255) / 256), dim3(256), 0,
                     (hipStream_t)stream, c->state, c->batch);
  SVLA_CHECK_LAUNCH();
  return SVLA_OK;
}

int svla_kv_append_bf16(const svla_kv_cache* c, const void* k, int ldk, long k_bs, const void* v,
                        int ldv, long v_bs, int rows, const int* counts, const int* at,
                        svla_stream_t stream) {
  if (!cache_ok(c) || rows < 0 || rows > kMaxPos) return SVLA_EINVAL;
  if (rows == 0 && !at) return SVLA_OK;
  if (rows > 0 && (!rows_ok(k, ldk, k_bs, c->n_kv_heads) || !rows_ok(v, ldv, v_bs, c->n_kv_heads)))
    return SVLA_EINVAL;
  AppendArgs a;
  a.c = device_cache(c);
  a.k = static_cast<const bf16*>(k); a.ldk = ldk; a.k_bs = k_bs;
  a.v = static_cast<const bf16*>(v); a.ldv = ldv; a.v_bs = v_bs;
  a.counts = counts;
  a.at = at;
  a.rows = rows;
  hipStream_t s = (hipStream_t)stream;
  // records that `rows` consecutive positions touch, at most
  long tiles = rows ? (rows + TOK - 2) / TOK + 1 + (c->sinks && rows > 1) : 1;
  tiles = min(tiles, (long)a.c.ring_tiles + a.c.sink_tiles);
  const long units = tiles * c->n_kv_heads;
  const size_t rec = c->format == SVLA_KV_MXFP4 ? kRec<4> : kRec<8>;
  // one workgroup per sequence up to 12 records (of 8 bits: 51 KB of LDS)
  const int waves = units <= 12 ? (int)units : 4;
  const dim3 grid((unsigned)min((units + waves - 1) / waves, 1L << 20), c->batch);
  if (c->format == SVLA_KV_MXFP4)
    hipLaunchKernelGGL(append_kernel<4>, grid, dim3(64 * waves), waves * rec, s, a);
  else
    hipLaunchKernelGGL(append_kernel<8>, grid, dim3(64 * waves), waves * rec, s, a);
  SVLA_CHECK_LAUNCH();
  if (grid.x > kMaxArrivals) {
    hipLaunchKernelGGL(advance_kernel, dim3((c->batch + 255) / 256), dim3(256), 0, s, a, c->batch);
    SVLA_CHECK_LAUNCH();
  }
  return SVLA_OK;
}

int svla_kv_read_bf16(const svla_kv_cache* c, void* k, int ldk, long k_bs, void* v, int ldv,
                      long v_bs, int start, const int* starts, int rows, svla_stream_t stream) {
  if (!cache_ok(c) || rows < 0 || rows > kMaxPos || (!starts && (start < 0 || start > kMaxPos)))
    return SVLA_EINVAL;
  if (rows == 0) return SVLA_OK;
  if (!rows_ok(k, ldk, k_bs, c->n_kv_heads) || !rows_ok(v, ldv, v_bs, c->n_kv_heads))
    return SVLA_EINVAL;
  ReadArgs a;
  a.c = device_cache(c);
  a.k = static_cast<bf16*>(k); a.ldk = ldk; a.k_bs = k_bs;
  a.v = static_cast<bf16*>(v); a.ldv = ldv; a.v_bs = v_bs;
  a.starts = starts;
  a.start = start;
  a.rows = rows;
  const long tiles = (rows + TOK - 2) / TOK + 1 + (c->sinks > 0);
  const dim3 grid((unsigned)min(tiles, 1L << 20), c->n_kv_heads, c->batch);
  if (c->format == SVLA_KV_MXFP4)
    hipLaunchKernelGGL(read_kernel<4>, grid, dim3(64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(read_kernel<8>, grid, dim3(64), 0, (hipStream_t)stream, a);
  SVLA_CHECK_LAUNCH();
  return SVLA_OK;
}

long svla_kv_attention_scratch(const svla_kv_cache* c, int rows, int hq, int window) {
  if (!cache_ok(c) || rows <= 0 || hq <= 0 || hq % c->n_kv_heads || window < 0) return 0;
  return scratch_of(c, plan_attend(c, rows, hq, window), rows, hq);
}

int svla_kv_step_bf16(const svla_kv_cache* c, const void* q, int ldq, long q_bs, const void* k,
                      int ldk, long k_bs, const void* v, int ldv, long v_bs, void* o, int ldo,
                      long o_bs, int rows, const int* counts, const int* at, int hq, float scale,
                      int window, void* scratch, long scratch_bytes, svla_stream_t stream) {
  Plan p;
  AttendArgs a;
  const int rc = attend_args(c, q, ldq, q_bs, o, ldo, o_bs, rows, counts, hq, scale, window, scratch,
                             scratch_bytes, &p, &a);
  if (rc) return rc;
  if (rows > 0 && (!rows_ok(k, ldk, k_bs, c->n_kv_heads) || !rows_ok(v, ldv, v_bs, c->n_kv_heads)))
    return SVLA_EINVAL;
  // One new row, and one workgroup for all the columns of its record: written
  // on the way (one token after 241 held: 6.3 us against 6.0 + 5.2 in two
  // launches; 32 sequences in windows of 4096: 15.1 + 4.4 against 7.4 + 16.9 + 4.3)
  if (rows != 1 || p.grid.x != 1) {
    const int w = svla_kv_append_bf16(c, k, ldk, k_bs, v, ldv, v_bs, rows, counts, at, stream);
    if (w || rows == 0) return w;
  } else {
    a.k = static_cast<const bf16*>(k); a.k_bs = k_bs;
    a.v = static_cast<const bf16*>(v); a.v_bs = v_bs;
    a.at = at;
  }
  return run_attend(c, p, a, (hipStream_t)stream);
}

int svla_kv_attention_bf16(const svla_kv_cache* c, const void* q, int ldq, long q_bs, void* o,
                           int ldo, long o_bs, int rows, const int* counts, int hq, float scale,
                           int window, void* scratch, long scratch_bytes, svla_stream_t stream) {
  Plan p;
  AttendArgs a;
  const int rc = attend_args(c, q, ldq, q_bs, o, ldo, o_bs, rows, counts, hq, scale, window, scratch,
                             scratch_bytes, &p, &a);
  return rc || rows == 0 ? rc : run_attend(c, p, a, (hipStream_t)stream);
}

}  // extern "C"
