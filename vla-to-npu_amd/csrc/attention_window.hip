// Attention with a sliding window and sinks for gfx950 (head_dim 64): the query
// at position p = q_pos + row sees the keys of positions (p - window, p] and of
// the first `sinks` positions, of the lens[b] that its sequence has.
//
// o = sum_j p_j v_j / sum_j p_j over the visible keys, p_j = 2^(c s_j - c m):
// one pass over the keys with a running maximum m, rounded probabilities in
// both sums as in attention_kernel, whose tiles, operand order and LDS ring
// these are: a workgroup is 64 QT query rows of one head, 16 QT a wave, and
// streams blocks of 64 keys.
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
};

// Elements of 8 bf16 that are infinite or NaN: bit 15 / 31 of every dword
__device__ __forceinline__ u32x4 nonfinite(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ((w[i] & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
  return w;
}

template <int QT>
__global__ __launch_bounds__(256, 2) void window_kernel(WindowArgs p) {
  constexpr int QW = 16 * QT, BQ = 4 * QW;
  __shared__ __attribute__((aligned(1024))) bf16 sK0[BKEY * D], sK1[BKEY * D], sK2[BKEY * D];
  __shared__ __attribute__((aligned(1024))) bf16 sV0[BKEY * D], sV1[BKEY * D], sV2[BKEY * D];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.y, b = blockIdx.z;
  const int kvh = h * p.hkv / p.hq;
  const int q0 = blockIdx.x * BQ;
  const int grp = lane >> 4, col = lane & 15;
  const int qw = q0 + wave * QW;
  const bf16* qb = p.q + b * p.q_bs + h * D;
  const bf16* kb = p.k + b * p.k_bs + kvh * D;
  const bf16* vb = p.v + b * p.v_bs + kvh * D;
  const int len = p.lens ? min(max(p.lens[b], 0), p.sk) : p.sk;

  // blocks of 64 keys: those of the sinks, then those of the rows' windows
  const int pend = min(p.q_pos + min(p.sq, q0 + BQ), len);          // keys below it
  const int sink_blocks = (min(p.sinks, pend) + BKEY - 1) / BKEY;
  const int from = max(sink_blocks, max(p.q_pos + q0 - p.window + 1, 0) / BKEY);
  const int nb = sink_blocks + max((pend + BKEY - 1) / BKEY - from, 0);
  auto key0 = [&](int blk) { return (blk < sink_blocks ? blk : from + blk - sink_blocks) * BKEY; };

  long koff[2], voff[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int key = (wave * 2 + j) * 8 + (lane >> 3);
    const int c = (lane & 7) ^ (key & 7);
    koff[j] = (long)key * p.ldk + c * 8;
    voff[j] = (long)key * p.ldv + c * 8;
  }
  auto issue = [&](auto SI, int blk) {
    constexpr int S = decltype(SI)::value;
    bf16* sk = S == 0 ? sK0 : S == 1 ? sK1 : sK2;
    bf16* sv = S == 0 ? sV0 : S == 1 ? sV1 : sV2;
    const int k0 = key0(min(blk, nb - 1));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = (wave * 2 + j) * 8 + (lane >> 3);
      const int rows_left = p.sk - 1 - k0;
      const long adj = key > rows_left ? (long)(rows_left - key) : 0;
      const bf16* gk = kb + (long)k0 * p.ldk + koff[j] + adj * p.ldk;
      const bf16* gv = vb + (long)k0 * p.ldv + voff[j] + adj * p.ldv;
      __builtin_amdgcn_global_load_lds((void*)gk, (lds_ptr_t)(sk + (wave * 2 + j) * 512), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((void*)gv, (lds_ptr_t)(sv + (wave * 2 + j) * 512), 16, 0, 0);
    }
  };

  bf16x8 qf[QT][2];
  int qpos[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = min(qw + qt * 16 + col, p.sq - 1);
    qpos[qt] = p.q_pos + qi;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) qf[qt][ks] = ld8(qb + (long)qi * p.ldq + ks * 32 + grp * 8);
  }
  // positions of the wave's first and last row
  const int wlo = p.q_pos + min(qw, p.sq - 1), whi = p.q_pos + min(qw + QW, p.sq) - 1;

  f32x4 o[QT][5];
  float m_run[QT], m_thr[QT], m_off[QT];
  const float c = p.scale_log2;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
    for (int t = 0; t < 5; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[qt] = -INFINITY;
    m_thr[qt] = -INFINITY;
    m_off[qt] = 0.f;
  }
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = f2bf(1.0f);

  auto compute = [&](auto SI, int blk) {
    constexpr int S = decltype(SI)::value;
    const bf16* sk = S == 0 ? sK0 : S == 1 ? sK1 : sK2;
    const bf16* sv = S == 0 ? sV0 : S == 1 ? sV1 : sV2;
    const int k0 = key0(blk);
    if (qw >= p.sq || k0 > whi || (k0 + BKEY - 1 <= wlo - p.window && k0 >= p.sinks)) return;
    const bool full = k0 + BKEY - 1 <= wlo && k0 + BKEY <= len &&
                      (k0 > whi - p.window || k0 + BKEY <= p.sinks);
    auto sees = [&](int qt, int key) {
      return key <= qpos[qt] && key < len && (key > qpos[qt] - p.window || key < p.sinks);
    };
    f32x4 sacc[4][QT];
#pragma unroll
    for (int ts = 0; ts < 4; ++ts) {
      bf16x8 kf[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        kf[ks] = *reinterpret_cast<const bf16x8*>(&sk[kv_off(ts * 16 + col, ks * 32 + grp * 8)]);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[ks], qf[qt][ks], a, 0, 0, 0);
        sacc[ts][qt] = a;
      }
    }
    bf16x8 pf[QT][2];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (!full) {
#pragma unroll
        for (int ts = 0; ts < 4; ++ts)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sacc[ts][qt][i] = sees(qt, k0 + ts * 16 + grp * 4 + i) ? sacc[ts][qt][i] : -INFINITY;
      }
      float mx = sacc[0][qt][0];
#pragma unroll
      for (int ts = 0; ts < 4; ++ts)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = smax(mx, sacc[ts][qt][i]);
      mx = max_xor32(max_xor16(mx));
      // the maximum moves only when a score passes it by 2^8 (attention_kernel)
      const bool grow = mx * c > m_thr[qt];
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float m_new = smax(m_run[qt], mx);
        const float alpha = m_run[qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run[qt] - m_new) * c);
#pragma unroll
        for (int t = 0; t < 5; ++t) o[qt][t] *= alpha;
        m_run[qt] = m_new;
        m_thr[qt] = m_new * c + 8.f;
        m_off[qt] = -((m_new == -INFINITY ? 0.f : m_new) * c);
      }
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 vf[4];
#pragma unroll
      for (int td = 0; td < 4; ++td) {
        const v4i16 lo = v_tr_read(sv, kk * 32 + 4 * grp, td * 16, col);
        const v4i16 hi = v_tr_read(sv, kk * 32 + 16 + 4 * grp, td * 16, col);
        const v4i16 w8[2] = {lo, hi};
        vf[td] = *reinterpret_cast<const bf16x8*>(w8);
      }
      // A row must not meet what it does not see, not even as 0 * NaN: where a
      // block has keys that some row does not see and V holds infinities or
      // NaNs, those are taken out of V and added to the rows that see them,
      // found by products of indicators.
      if (!full) {
        u32x4 bad[4];
        unsigned some = 0;
#pragma unroll
        for (int td = 0; td < 4; ++td) {
          bad[td] = nonfinite(__builtin_bit_cast(u32x4, vf[td]));
          some |= bad[td][0] | bad[td][1] | bad[td][2] | bad[td][3];
        }
        if (__builtin_amdgcn_ballot_w64(some != 0)) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            bf16x8 vis;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              vis[j] = f2bf(sees(qt, k0 + kk * 32 + (j >> 2) * 16 + grp * 4 + (j & 3)) ? 1.f : 0.f);
#pragma unroll
            for (int td = 0; td < 4; ++td)
#pragma unroll
              for (int what = 0; what < 3; ++what) {   // +inf, -inf, NaN
                bf16x8 hit;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float x = bf2f(vf[td][j]);
                  const bool is = what == 0 ? x == INFINITY : what == 1 ? x == -INFINITY : x != x;
                  hit[j] = f2bf(is ? 1.f : 0.f);
                }
                f32x4 cnt = {0.f, 0.f, 0.f, 0.f};
                cnt = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hit, vis, cnt, 0, 0, 0);
                const float add = what == 0 ? INFINITY : what == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
                for (int i = 0; i < 4; ++i) o[qt][td][i] += cnt[i] > 0.f ? add : 0.f;
              }
          }
#pragma unroll
          for (int td = 0; td < 4; ++td) {
            u32x4 w = __builtin_bit_cast(u32x4, vf[td]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] &= ((bad[td][i] & 0x8000u) ? 0u : 0xffffu) | ((bad[td][i] >> 31) ? 0u : 0xffff0000u);
            vf[td] = __builtin_bit_cast(bf16x8, w);
          }
        }
      }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pf[qt][kk][hh * 4 + i] =
                f2bf(__builtin_amdgcn_exp2f(__builtin_fmaf(sacc[2 * kk + hh][qt][i], c, m_off[qt])));
#pragma unroll
        for (int td = 0; td < 4; ++td)
          o[qt][td] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[td], pf[qt][kk], o[qt][td], 0, 0, 0);
        o[qt][4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[qt][kk], o[qt][4], 0, 0, 0);
      }
    }
  };

  // Before each barrier: vmcnt(4), the next stage's 4 DMA instructions stay in
  // flight, and lgkmcnt(0), this wave's reads of the stage that the DMA issued
  // right after the barrier refills are done.
  auto sync_step = [&]() __attribute__((always_inline)) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x074);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  __builtin_amdgcn_s_waitcnt(0xF70);   // Q is here before the DMA prologue
  if (nb > 0) {                        // uniform across the workgroup
    issue(I0{}, 0);
    issue(I1{}, 1);
    for (int blk = 0; blk < nb; blk += 3) {
      sync_step();
      issue(I2{}, blk + 2);
      compute(I0{}, blk);
      if (blk + 1 >= nb) break;
      sync_step();
      issue(I0{}, blk + 3);
      compute(I1{}, blk + 1);
      if (blk + 2 >= nb) break;
      sync_step();
      issue(I1{}, blk + 4);
      compute(I2{}, blk + 2);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);       // no DMA into LDS outlives the workgroup

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
  if (sq <= 64 || g2 < 512)
    hipLaunchKernelGGL(window_kernel<1>, dim3((sq + 63) / 64, hq, batch), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL(window_kernel<2>, dim3((sq + 127) / 128, hq, batch), dim3(256), 0, s, p);
  SVLA_CHECK_LAUNCH();
  return SVLA_OK;
}
