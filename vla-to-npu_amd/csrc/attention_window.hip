// Attention with a sliding window and sinks for gfx950 (head_dim 64): the query
// at position p = q_pos + row sees the keys of positions (p - window, p] and of
// the first `sinks` positions, of the lens[b] that its sequence has.
//
// o = sum_j p_j v_j / sum_j p_j over the visible keys, p_j = 2^(c s_j - c m), in
// one pass over the keys, for any reference m (0 but for the second time, see
// the kernel), with the rounded probabilities in both sums.  Tiles and operand
// order are attention_kernel's: a workgroup is 64 QT query rows of one head,
// 16 QT a wave, and goes through the blocks of 64 keys that some row sees.
//
// MI355X: 2 x 16384 rows of 15 heads, window 4096, 593 to 610 us (451 GFLOP, 740
// to 760 TFLOP/s, half of a large library product's 1490).  With 128 rows a
// workgroup and three waves per SIMD a block of 64 keys and 32 rows takes 1470
// cycles, of which 36 MFMAs are 576 and the vector instructions 620.  Measured
// and not kept: the next scores beside the last products in one instruction
// stream (639 us against 606: two waves per SIMD; in another run 711, of which
// timing copies without the exponentials took 622 and without staging and
// barriers 571: no one pipe bounds it), 256 rows (635), 64 rows (722).  8 x 2000 rows of 12 heads, window 500, 57 to 62 us (86 MB, 17.9
// GFLOP): 10 blocks a workgroup, 4 of them cut by the window's ends; window 64
// takes 37 us (98 MB).
#include "attention_tile.h"

namespace {

struct WindowArgs {
  const bf16* q; long ldq, q_bs;
  const bf16* k; long ldk, k_bs;
  const bf16* v; long ldv, v_bs;
  bf16* o; long ldo, o_bs;
  const int* lens;
  int sq, sk, hq, hkv, q_pos, window, sinks;
  float scale_log2;
  int row_blocks, blocks, run;          // of a KV head, of the call, dealt at a time
};

// Elements of 8 bf16 that are infinite or NaN: bit 15 / 31 of every dword
__device__ __forceinline__ u32x4 nonfinite(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ((w[i] & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
  return w;
}

// The loop: blocks of 64 keys go through registers into two LDS stages, so that
// a block's loads have the whole of the block before them to arrive.
template <int QT>
__global__ __launch_bounds__(256, QT == 2 ? 3 : 4) void window_kernel(WindowArgs p) {
  constexpr int QW = 16 * QT, BQ = 4 * QW;
  // K of two stages, then V of two: 8 KB each
  constexpr int STAGE = BKEY * D * 2, V_AT = 2 * STAGE;
  __shared__ __attribute__((aligned(1024))) char lds[4 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroup i runs on XCD i % 8.  The row blocks of all (sequence, KV head)s
  // are dealt to the XCDs in runs of `run`, all query heads of a block in a
  // row, so that what one XCD works on at a time shares keys in its L2.
  const int group = p.hq / p.hkv;
  const unsigned slot = blockIdx.x >> 3;
  const unsigned in_run = slot % (p.run * group);
  const unsigned blk_id = (slot / (p.run * group) * 8 + (blockIdx.x & 7)) * p.run + in_run / group;
  if (blk_id >= (unsigned)p.blocks) return;
  const int bk = blk_id / p.row_blocks;            // (sequence, KV head)
  const int b = bk / p.hkv, kvh = bk - b * p.hkv;
  const int h = kvh * group + in_run % group;
  const int q0 = (blk_id - bk * p.row_blocks) * BQ;
  const int grp = lane >> 4, col = lane & 15;
  const int qw = q0 + wave * QW;
  const bf16* kb = p.k + b * p.k_bs + kvh * D;
  const bf16* vb = p.v + b * p.v_bs + kvh * D;
  const int len = p.lens ? min(max(p.lens[b], 0), p.sk) : p.sk;

  // blocks of 64 keys: those of the sinks, then those of the rows' windows
  const int pend = min(p.q_pos + min(p.sq, q0 + BQ), len);          // keys below it
  const int sink_blocks = (min(p.sinks, pend) + BKEY - 1) / BKEY;
  const int from = max(sink_blocks, max(p.q_pos + q0 - p.window + 1, 0) / BKEY);
  const int nb = sink_blocks + max((pend + BKEY - 1) / BKEY - from, 0);
  auto key0 = [&](int blk) { return (blk < sink_blocks ? blk : from + blk - sink_blocks) * BKEY; };

  // rows tid / 8 and 32 + tid / 8 of a block, 16 bytes each (rows past the last
  // key repeat it: never seen)
  u32x4 rk[2], rv[2];
  const int srow = tid >> 3, schunk = (tid & 7) * 8;
  const unsigned kstep = 2u * p.ldk, vstep = 2u * p.ldv;           // bytes of a row
  const unsigned kvo = srow * kstep + schunk * 2, vvo = srow * vstep + schunk * 2;
  const char *gk, *gv;                 // block `next`
  int next, next_key;
  auto start = [&]() {
    next = 0;
    next_key = key0(0);
    gk = (const char*)(kb + (long)next_key * p.ldk);
    gv = (const char*)(vb + (long)next_key * p.ldv);
  };
  auto load = [&]() __attribute__((always_inline)) {
    if (next_key + BKEY <= p.sk) {
      rk[0] = *(const u32x4*)(gk + kvo);
      rk[1] = *(const u32x4*)(gk + 32 * kstep + kvo);
      rv[0] = *(const u32x4*)(gv + vvo);
      rv[1] = *(const u32x4*)(gv + 32 * vstep + vvo);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned r = min(srow + 32 * i, p.sk - 1 - next_key);
        rk[i] = *(const u32x4*)(gk + (r * kstep + schunk * 2));
        rv[i] = *(const u32x4*)(gv + (r * vstep + schunk * 2));
      }
    }
    // (past the last block: that one again, never used)
    if (++next < nb) {
      const int step = next == sink_blocks ? (from - sink_blocks + 1) * BKEY : BKEY;
      next_key += step;
      gk += (long)step * kstep;
      gv += (long)step * vstep;
    } else {
      next = nb - 1;
    }
  };
  int sofs = 2 * kv_off(srow, schunk);
  auto store = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *(u32x4*)(lds + sofs + 32 * i * D * 2) = rk[i];
      *(u32x4*)(lds + sofs + V_AT + 32 * i * D * 2) = rv[i];
    }
    sofs ^= STAGE;
  };

  bf16x8 qf[QT][2];
  int last[QT], before[QT];       // keys of this lane's row: (before, last] and sinks
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = min(qw + qt * 16 + col, p.sq - 1);
    last[qt] = min(p.q_pos + qi, len - 1);
    before[qt] = p.q_pos + qi - p.window;
    const bf16* q = p.q + b * p.q_bs + (long)qi * p.ldq + h * D;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) qf[qt][ks] = ld8(q + ks * 32 + grp * 8);
  }
  // positions of the wave's first and last row
  const int wlo = p.q_pos + min(qw, p.sq - 1), whi = p.q_pos + min(qw + QW, p.sq) - 1;

  f32x4 o[QT][5];
  float m_run[QT], m_off[QT];
  const float c = p.scale_log2;
  auto clear = [&](float m) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
      for (int t = 0; t < 5; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[qt] = m;
      m_off[qt] = 0.f;
    }
  };
  clear(0.f);
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = f2bf(1.0f);
  int track = 0;           // the second time over the keys

  // Byte offsets of the lane's operand reads within a stage (kv_off: a key's row
  // is 128 bytes, its 16-byte chunks are swapped by the key's low bits, which
  // steps of 16 keys keep).
  int kofs[2], vofs[4];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) kofs[ks] = 2 * kv_off(col, ks * 32 + grp * 8);
#pragma unroll
  for (int td = 0; td < 4; ++td) vofs[td] = 2 * kv_off(4 * grp + (col >> 2), td * 16 + 4 * (col & 3));

  auto sees = [&](int qt, int key) {
    return key <= last[qt] && (key > before[qt] || key < p.sinks);
  };
  f32x4 sacc[2][QT];
  bf16x8 vf[4];
  auto v_frag = [&](int hf, int td) __attribute__((always_inline)) {
    const char* at = lds + vofs[td] + (V_AT + hf * 32 * D * 2);
    const v4i16 w8[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)at),
                         __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(at + 16 * D * 2))};
    return *reinterpret_cast<const bf16x8*>(w8);
  };
  // scores of half hf of the block, and its V
  auto score = [&](int hf) __attribute__((always_inline)) {
#pragma unroll
    for (int ts = 0; ts < 2; ++ts) {
      bf16x8 kf[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        kf[ks] = *reinterpret_cast<const bf16x8*>(lds + kofs[ks] + (hf * 2 + ts) * 16 * D * 2);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[ks], qf[qt][ks], a, 0, 0, 0);
        sacc[ts][qt] = a;
      }
    }
#pragma unroll
    for (int td = 0; td < 4; ++td) vf[td] = v_frag(hf, td);
  };
  // Masks the scores of the keys k0 .. k0 + 31: of (before, last] and the sinks
  // the row's own are left.
  auto mask = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int at = k0 + grp * 4 - before[qt] - 1, n = max(last[qt] - before[qt], 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = (i >> 2) * 16 + (i & 3);
        bool in = (unsigned)(at + key) < (unsigned)n;
        if (k0 < p.sinks) in = sees(qt, k0 + grp * 4 + key);
        sacc[i >> 2][qt][i & 3] = in ? sacc[i >> 2][qt][i & 3] : -INFINITY;
      }
    }
  };
  // Follows the maximum, which moves only when a score passes it by 2^8 as in
  // attention_kernel.
  auto follow = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float mx = sacc[0][qt][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = smax(mx, sacc[i >> 2][qt][i & 3]);
      mx = max_xor32(max_xor16(mx));
      const bool grow = mx * c > m_run[qt] * c + 8.f;
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float m_new = smax(m_run[qt], mx);
        const float alpha = m_run[qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[qt] - m_new) * c);
#pragma unroll
        for (int t = 0; t < 5; ++t) o[qt][t] *= alpha;
        m_run[qt] = m_new;
        m_off[qt] = -((m_new == -INFINITY ? 0.f : m_new) * c);
      }
    }
  };
  // Takes infinities and NaNs out of V; returns whether there were any.
  auto take_out = [&]() __attribute__((always_inline)) {
    unsigned some = 0;
#pragma unroll
    for (int td = 0; td < 4; ++td) {
      u32x4 w = __builtin_bit_cast(u32x4, vf[td]);
      const u32x4 bad = nonfinite(w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        some |= bad[i];
        w[i] &= ~((bad[i] >> 15) * 0xffffu);
      }
      vf[td] = __builtin_bit_cast(bf16x8, w);
    }
    return __builtin_amdgcn_ballot_w64(some != 0) != 0;
  };
  auto accumulate = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      bf16x8 pf;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        pf[i] = f2bf(__builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i >> 2][qt][i & 3], c, m_off[qt])));
#pragma unroll
      for (int td = 0; td < 4; ++td)
        o[qt][td] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[td], pf, o[qt][td], 0, 0, 0);
      o[qt][4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf, o[qt][4], 0, 0, 0);
    }
  };
  // Gives them to the rows that see them: how often each row sees +inf, -inf and
  // NaN in each depth of the V of keys k0 .. k0 + 31, as products of indicators.
  auto put_back = [&](int hf, int k0) __attribute__((always_inline)) {
#pragma unroll 1
    for (int it = 0; it < 12; ++it) {
      const int td = it / 3, what = it % 3;
      const bf16x8 x = td < 2 ? (td == 0 ? v_frag(hf, 0) : v_frag(hf, 1))
                              : (td == 2 ? v_frag(hf, 2) : v_frag(hf, 3));
      const float add = what == 0 ? INFINITY : what == 1 ? -INFINITY : __builtin_nanf("");
      bf16x8 hit;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = bf2f(x[j]);
        hit[j] = f2bf((what == 2 ? y != y : y == add) ? 1.f : 0.f);
      }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        bf16x8 vis;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          vis[j] = f2bf(sees(qt, k0 + (j >> 2) * 16 + grp * 4 + (j & 3)) ? 1.f : 0.f);
        f32x4 cnt = {0.f, 0.f, 0.f, 0.f};
        cnt = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hit, vis, cnt, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[qt][t][i] += t == td && cnt[i] > 0.f ? add : 0.f;
      }
    }
  };

  // lgkmcnt(0): this wave's reads of the stage that is written next, and its own
  // writes, are done; loads into registers stay in flight
  auto sync_step = [&]() __attribute__((always_inline)) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  // Softmax needs no maximum where exp(s) itself neither over- nor underflows:
  // any reference gives the same quotient, and bf16 keeps fp32's range.  So the
  // first time over the keys takes the reference 0.  Where a row's sum leaves
  // [2^-40, 2^100], or an output 2^100 (also by infinities and NaNs, even from
  // behind the mask, as 0 * NaN), the workgroup goes over its keys once more,
  // following the maximum, and a row then meets only what it sees, infinities
  // and NaNs apart.
  // The wave's blocks in the list: [see0, see1) of the windows' blocks hold keys
  // that some row sees, [full0, full1) only keys that all do; of the sinks' the
  // first sink_full.
  const int shift = sink_blocks - from;
  const int see0 = max(max(wlo - p.window + 1, 0) / BKEY + shift, sink_blocks);
  const int see1 = qw < p.sq ? min(whi / BKEY + 1 + shift, nb) : 0;
  const int full0 = (max(whi - p.window + 1, 0) + BKEY - 1) / BKEY + shift;
  const int full1 = min(wlo + 1, len) / BKEY + shift;
  const int sink_full = min(min(wlo + 1, len), p.sinks) / BKEY;
  const int sink_see = qw < p.sq ? sink_blocks : 0;
  for (;;) {
    if (nb > 0) {                      // uniform across the workgroup
      start();
      load();
      const u32x4 k0 = rk[0], k1 = rk[1], v0 = rv[0], v1 = rv[1];
      load();                          // two blocks on their way
      const u32x4 k2 = rk[0], k3 = rk[1], v2 = rv[0], v3 = rv[1];
      rk[0] = k0; rk[1] = k1; rv[0] = v0; rv[1] = v1;
      store();
      rk[0] = k2; rk[1] = k3; rv[0] = v2; rv[1] = v3;
      sync_step();
    }
    for (int blk = 0; blk < nb; ++blk) {
      asm volatile("" : "+s"(track));  // one loop for both
      store();                         // (the last block's again behind it)
      load();
      const bool is_sink = blk < sink_blocks;
      if (is_sink ? blk < sink_see : blk >= see0 && blk < see1) {
        const bool part = is_sink ? blk >= sink_full : blk < full0 || blk >= full1;
        const int k0 = key0(blk), k1 = k0 + 32;
        bool odd = false;
        score(0);
        if (part) mask(k0);
        if (track) {
          follow();
          odd = take_out();
        }
        accumulate();
        if (track && odd) put_back(0, k0);
        score(1);
        if (part) {
          if (!(k1 <= whi && k1 < len && (k1 + 31 > wlo - p.window || k1 < p.sinks))) goto done;
          mask(k1);
        }
        if (track) {
          follow();
          odd = take_out();
        }
        accumulate();
        if (track && odd) put_back(1, k1);
      }
    done:
#pragma unroll
      for (int i = 0; i < 2; ++i) kofs[i] ^= STAGE;
#pragma unroll
      for (int i = 0; i < 4; ++i) vofs[i] ^= STAGE;
      sync_step();
    }
    bool bad = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float top = o[qt][4][0];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = smax(top, fabsf(o[qt][t][i]));
      const bool sees_some = last[qt] > max(before[qt], -1) || (p.sinks > 0 && last[qt] >= 0);
      bad |= sees_some && !(top < 0x1p100f && o[qt][4][0] >= 0x1p-40f);
    }
    if (track || !__syncthreads_or(bad && qw < p.sq)) break;
    track = 1;
    clear(-INFINITY);
    // back to the first stage
    if (nb & 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) kofs[i] ^= STAGE;
#pragma unroll
      for (int i = 0; i < 4; ++i) vofs[i] ^= STAGE;
    } else {
      sofs ^= STAGE;
    }
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = qw + qt * 16 + col;
    if (qi >= p.sq) continue;
    const float l = o[qt][4][0];
    const float inv = l > 0.f ? 1.0f / l : l;    // nothing visible: 0; NaN stays
    bf16* orow = p.o + b * p.o_bs + (long)qi * p.ldo + h * D;
#pragma unroll
    for (int td = 0; td < 4; ++td) {
      bf16x4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = f2bf(o[qt][td][i] * inv);
      *reinterpret_cast<bf16x4*>(orow + td * 16 + grp * 4) = r;
    }
  }
}

}  // namespace

extern "C" int svla_attention_window_bf16(const void* q, int ldq, long q_bs, const void* k,
                                          int ldk, long k_bs, const void* v, int ldv, long v_bs,
                                          void* o, int ldo, long o_bs, int batch, int sq, int sk,
                                          int hq, int hkv, int head_dim, float scale, int q_pos,
                                          const int* lens, int window, int sinks,
                                          svla_stream_t stream) {
  constexpr int kMax = 1 << 30;
  if (head_dim != D || hq <= 0 || hkv <= 0 || hq % hkv || sq < 0 || sk <= 0 || batch < 0 ||
      hq > 65535 || batch > 65535 || sq > kMax || sk > kMax)
    return SVLA_EINVAL;
  if (window < 1 || sinks < 0 || q_pos < 0 || q_pos > kMax - sq || !(scale > 0.f) || !(scale < 1e30f))
    return SVLA_EINVAL;
  if (ldq % 8 || ldk % 8 || ldv % 8 || ldo % 4 || q_bs % 8 || k_bs % 8 || v_bs % 8 || o_bs % 4)
    return SVLA_EINVAL;
  if (ldk > (1 << 24) || ldv > (1 << 24)) return SVLA_EINVAL;   // offsets within a block: 32 bits
  if (ldq < hq * D || ldk < hkv * D || ldv < hkv * D || ldo < hq * D) return SVLA_EINVAL;
  if (!svla_aligned16(q) || !svla_aligned16(k) || !svla_aligned16(v) || ((uintptr_t)o & 7))
    return SVLA_EINVAL;
  if (sq == 0 || batch == 0) return SVLA_OK;
  if (!q || !k || !v || !o) return SVLA_EINVAL;
  WindowArgs p;
  p.q = static_cast<const bf16*>(q); p.ldq = ldq; p.q_bs = q_bs;
  p.k = static_cast<const bf16*>(k); p.ldk = ldk; p.k_bs = k_bs;
  p.v = static_cast<const bf16*>(v); p.ldv = ldv; p.v_bs = v_bs;
  p.o = static_cast<bf16*>(o); p.ldo = ldo; p.o_bs = o_bs;
  p.lens = lens;
  p.sq = sq; p.sk = sk; p.hq = hq; p.hkv = hkv;
  p.q_pos = q_pos;
  p.window = min(window, kMax);
  p.sinks = min(sinks, kMax);
  p.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  const long g2 = (long)((sq + 127) / 128) * hq * batch;
  // 128 rows a workgroup share each key's LDS reads, 64 rows waste fewer keys at
  // the ends of a short window and fill more of the chip (MI355X, 64 / 128 rows:
  // 2 x 16384 x 15 heads, window 4096: 723 / 606 us; 8 x 2000 x 12, window 500:
  // 69 / 77)
  const int qt = g2 >= 512 && min(window, sk) >= 1024 ? 2 : 1;
  p.row_blocks = (sq + 64 * qt - 1) / (64 * qt);
  const long blocks = (long)p.row_blocks * hkv * batch;
  if (blocks > (1L << 24)) return SVLA_EINVAL;
  p.blocks = (int)blocks;
  p.run = (int)max(1L, min(16L, blocks / 32));
  const long runs = (blocks + p.run - 1) / p.run;
  const long grid = (runs + 7) / 8 * 8 * p.run * (hq / hkv);
  if (grid > 0x7fffffffL) return SVLA_EINVAL;
  if (qt == 1) hipLaunchKernelGGL(window_kernel<1>, dim3(grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(window_kernel<2>, dim3(grid), dim3(256), 0, s, p);
  SVLA_CHECK_LAUNCH();
  return SVLA_OK;
}
