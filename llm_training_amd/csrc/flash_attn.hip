// Launches of the flash attention kernels (flash_attn_kernels.h) on plain scores; flash_attn_mod_fwd.hip, _dq.hip and
// _dkdv.hip launch them on capped or biased scores and prefix masks.
#include "flash_attn_kernels.h"

namespace llmt {

// RoPE outside the attention kernels, for the launch paths without the fused form (dropout, the generic
// kernels, opt-in variants): strided [B, S, H, D] rows x -> y (y may alias x), one thread per 8 pairs
__global__ __launch_bounds__(256) void rope_bshd_kernel(AttnArgs a, const bf16* x, int x_sb, int x_ss, int x_sh, bf16* y,
                                                        int y_sb, int y_ss, int y_sh, int H, int D, float sign) {
  const int G = D / 16, half = D / 2;
  const int64_t n = (int64_t)a.B * a.S * H * G;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int g = (int)(e % G);
    int64_t t = e / G;
    const int h = (int)(t % H);
    t /= H;
    const int s = (int)(t % a.S), b = (int)(t / a.S);
    const int p = rope_pos(a, b, s);
    const float* cr = a.rcos + (int64_t)p * half + 8 * g;
    const float* sr = a.rsin + (int64_t)p * half + 8 * g;
    const bf16* xr = x + (int64_t)b * x_sb + (int64_t)s * x_ss + (int64_t)h * x_sh + 8 * g;
    bf16* yr = y + (int64_t)b * y_sb + (int64_t)s * y_ss + (int64_t)h * y_sh + 8 * g;
    bfv8 lo = *reinterpret_cast<const bfv8*>(xr), hi = *reinterpret_cast<const bfv8*>(xr + half);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = cr[j], sn = sign * sr[j], x1 = (float)lo[j], x2 = (float)hi[j];
      lo[j] = (__bf16)(x1 * c - x2 * sn);
      hi[j] = (__bf16)(x2 * c + x1 * sn);
    }
    *reinterpret_cast<bfv8*>(yr) = lo;
    *reinterpret_cast<bfv8*>(yr + half) = hi;
  }
}

}  // namespace llmt

using namespace llmt;

// Kernel selection. One kernel family per pass and head dim (D = 64 / 96 / 128):
//   forward  fa_fwd3_kernel      (LDS-DMA K/V ring, fused Q rotation, range masks)
//   dQ       fa_bwd_dq3_kernel   (also computes delta and the per-tile row constants for the dK/dV pass)
//   dK/dV    fa_bwd_dkdv5_kernel (software-pipelined, one wave per SIMD, GQA heads looped in-kernel)
// plus the generic kernels (fa_fwd_kernel / fa_bwd_{delta,dq,dkdv}_kernel) for dropout and other head dims.
// Losing variants of earlier rounds (one-wave-per-SIMD hand-allocated forward / dK/dV, head chains, GQA head
// pairs, the un-pipelined dK/dV loop, the separate prep pass) were removed after their A/Bs
// (profiles/r5_attention_fwd4.md, r5_dkdv6.md, r3_attention_head_pairs_ab.jsonl, r4_negative_probes.jsonl).
// Knobs, read per launch (recorded by ops/native.py llmt_env() into run metadata):
//   LLMT_FA_GENERIC=1     the generic kernels for every launch on plain scores (numerics reference);
//   LLMT_FA_RANGE_MASK=0  per-element mask compares instead of range masks, plain scores only (A/B reference);
//   LLMT_FA_EARLY_DMA=0   row loads before the first ring tiles in the prologues (A/B reference);
//   LLMT_FA_BMAJOR=0      batch-interleaved block order of dense rows (A/B reference; B4 S8192 Hq32 Hkv8 with
//                         the default batch-major order: forward 2.102 -> 2.068 ms, backward 7.795 -> 7.732 ms).
static int env_int(const char* name, int dflt) {
  const char* e = getenv(name);
  return e ? atoi(e) : dflt;
}
static bool generic_only() { return env_int("LLMT_FA_GENERIC", 0) == 1; }
static int range_masks() { return env_int("LLMT_FA_RANGE_MASK", 1); }
static int early_dma() { return env_int("LLMT_FA_EARLY_DMA", 1); }
static int bmajor_order() { return env_int("LLMT_FA_BMAJOR", 1); }
#ifdef LLMT_DIAG
static int attn_probe() { return env_int("LLMT_FA_PROBE", 0); }
#else
static int attn_probe() { return 0; }
#endif

// 1 in the diagnostic library (probes compiled in), 0 in the production one
extern "C" int llmt_attn_diag_build() {
#ifdef LLMT_DIAG
  return 1;
#else
  return 0;
#endif
}

static void set_dropout(AttnArgs& a, float p, uint32_t seed) {
  if (p <= 0.f) {
    a.drop_thresh = 0;
    return;
  }
  const double t = (double)p * 4294967296.0;
  a.drop_thresh = (uint32_t)(t >= 4294967295.0 ? 4294967295.0 : (t < 1.0 ? 1.0 : t));
  a.drop_seed = seed;
  a.drop_scale = 1.f / (1.f - p);
}

// buffer-load offsets are 32-bit: every row of one (batch, head) slice must be addressable
static bool fits32(int64_t S, int64_t row_stride) { return S * row_stride * 2 < 0x7fffffffLL; }
static bool strides32(std::initializer_list<int64_t> xs) {
  for (int64_t x : xs)
    if (x < 0 || x >= 0x7fffffffLL) return false;
  return true;
}

static bool aligned16(const void* p, int64_t s0, int64_t s1, int64_t s2) {
  return ((reinterpret_cast<uintptr_t>(p) & 15) == 0) && (s0 % 8 == 0) && (s1 % 8 == 0) && (s2 % 8 == 0);
}

// fused-RoPE arguments (AttnArgs::rpos ...); qrot: contiguous [B, S, Hq, D] scratch for rotated queries
static void set_rope(AttnArgs& a, const void* rpos, int rpos64, int64_t rp_sb, int64_t rp_ss, const float* rcos,
                     const float* rsin, int64_t rP, void* qrot, int D) {
  a.rpos = rpos; a.rpos64 = rpos64; a.rp_sb = (int)rp_sb; a.rp_ss = (int)rp_ss;
  a.rcos = rcos; a.rsin = rsin; a.rP = (int)rP;
  a.qrot = (bf16*)qrot;
  a.qr_sh = D; a.qr_ss = a.Hq * D; a.qr_sb = a.S * a.Hq * D;
}
static void rope_launch(const AttnArgs& a, const bf16* x, int x_sb, int x_ss, int x_sh, bf16* y, int y_sb, int y_ss,
                        int y_sh, int H, int D, float sign, hipStream_t stream) {
  const int64_t n = (int64_t)a.B * a.S * H * (D / 16);
  rope_bshd_kernel<<<stream_grid(n, 256), 256, 0, stream>>>(a, x, x_sb, x_ss, x_sh, y, y_sb, y_ss, y_sh, H, D, sign);
}
// the rotated queries in qrot become the kernels' q
static void use_qrot(AttnArgs& a) {
  a.q = a.qrot; a.q_sb = a.qr_sb; a.q_ss = a.qr_ss; a.q_sh = a.qr_sh;
}
static bool rope_ok(const void* rpos, const float* rcos, const float* rsin, int64_t rP, int64_t rp_sb, int64_t rp_ss) {
  if (!rcos) return rpos == nullptr && rsin == nullptr;
  return rsin && rP > 0 && rP < 0x7fffffffLL && ((reinterpret_cast<uintptr_t>(rcos) | reinterpret_cast<uintptr_t>(rsin)) & 15) == 0 &&
         strides32({rp_sb, rp_ss});
}

// Modified scores: `softcap` > 0 caps, `slopes` bias, `pend` prefix ends (see AttnArgs). False: not servable.
static bool set_mod(AttnArgs& a, float softcap, const float* slopes, const int* pend, void* olo) {
  if (!(softcap >= 0.f) || (pend && !a.causal)) return false;
  a.slopes = slopes;
  a.pend = pend;
  a.olo = (bf16*)olo;
  if (softcap > 0.f) {
    a.cap_k = 2.f * kLog2e * a.scale / softcap;
    a.cap_z = softcap * kLog2e;
    const double k = (double)a.scale / softcap, z = (double)a.scale * kLog2e, k2 = k * k, q3 = -0.0444022261 * z * k2 * k2 * k2;
    a.cap_q0 = (float)(0.999999456 * z);
    a.cap_q1 = (float)(-0.333263179 * z * k2);
    a.cap_q2 = (float)(0.131902966 * z * k2 * k2);
    a.cap_q3 = (float)q3;
    // (not where a coefficient leaves fp32's normal range)
    a.cap_x = fabs(q3) > 1e-36 && fabs(q3) < 1e36 ? (float)(0.5 / fabs(k)) : -1.f;
  }
  // range masks need run bounds with segment ids; dropout and fused rotations have no modified form
  return mod_of(a) == 0 || ((a.seg == nullptr || a.rs != nullptr) && !a.drop_thresh && !a.rcos);
}

// does the forward launch for this problem go to fa_fwd3_kernel (the kernel with the fused Q rotation)?
static bool fwd_uses_fwd3(int D, bool drop) { return !drop && !generic_only() && (D == 64 || D == 96 || D == 128); }

extern "C" hipError_t llmt_flash_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                                          const int* seg, int B, int S, int Hq, int Hkv, int D, int64_t q_sb,
                                          int64_t q_ss, int64_t q_sh, int64_t k_sb, int64_t k_ss, int64_t k_sh,
                                          int64_t v_sb, int64_t v_ss, int64_t v_sh, int64_t o_sb, int64_t o_ss,
                                          int64_t o_sh, float scale, int causal, int window, int seg_runs,
                                          float drop_p, uint32_t drop_seed, const void* rpos, int rpos64,
                                          int64_t rp_sb, int64_t rp_ss, const float* rcos, const float* rsin,
                                          int64_t rP, void* qrot, float softcap, const float* slopes,
                                          const int* pend, void* olo, hipStream_t stream) {
  if (Hkv <= 0 || Hq % Hkv) return hipErrorInvalidValue;
  if (!aligned16(q, q_sb, q_ss, q_sh) || !aligned16(k, k_sb, k_ss, k_sh) || !aligned16(v, v_sb, v_ss, v_sh) ||
      !aligned16(o, o_sb, o_ss, o_sh))
    return hipErrorInvalidValue;
  if (!rope_ok(rpos, rcos, rsin, rP, rp_sb, rp_ss)) return hipErrorInvalidValue;
  const bool rope = rcos != nullptr;
  if (!(drop_p >= 0.f && drop_p < 1.f)) return hipErrorInvalidValue;
  if (B == 0 || S == 0) return hipSuccess;
  if (!fits32(S, q_ss) || !fits32(S, k_ss) || !fits32(S, v_ss)) return hipErrorInvalidValue;
  if (!strides32({q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh})) return hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const bf16*)q; a.k = (const bf16*)k; a.v = (const bf16*)v; a.out = (bf16*)o; a.lse = lse; a.seg = seg;
  if (seg && seg_runs) {
    a.rs = seg + (int64_t)B * S;
    a.re = seg + 2 * (int64_t)B * S;
    if (seg_runs == 2) {  // + the work orders of the query / key blocks
      a.qord = seg + 3 * (int64_t)B * S;
      a.kord = a.qord + (int64_t)B * ((S + 127) / 128);
    }
  }
  a.B = B; a.S = S; a.Hq = Hq; a.Hkv = Hkv;
  a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh; a.k_sb = k_sb; a.k_ss = k_ss; a.k_sh = k_sh;
  a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh; a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
  a.scale = scale; a.causal = causal; a.window = window;
  set_dropout(a, drop_p, drop_seed);
  a.bmajor = bmajor_order();
  a.rmask = range_masks() && (seg == nullptr || a.rs != nullptr);
  a.early = early_dma();
  a.probe = attn_probe();
  if (rope) set_rope(a, rpos, rpos64, rp_sb, rp_ss, rcos, rsin, rP, qrot, D);
  if (!set_mod(a, softcap, slopes, pend, olo)) return hipErrorInvalidValue;
  if (const int mod = mod_of(a))
    return !aligned16(olo, 0, 0, 0) ? hipErrorInvalidValue
                                   : launch_mod_fwd(a, D, mod, (unsigned)((S + 127) / 128 * Hq * B), stream);
  const bool v3 = fwd_uses_fwd3(D, a.drop_thresh != 0);
  if (rope) {
    // fused RoPE: q holds unrotated queries (k is already rotated). fa_fwd3_kernel rotates its rows on load;
    // the generic kernel gets the rotated rows in the qrot scratch (q itself is never written)
    if (v3) {
      a.rope_q = 1;
    } else {
      if (!qrot) return hipErrorInvalidValue;
      rope_launch(a, a.q, a.q_sb, a.q_ss, a.q_sh, a.qrot, a.qr_sb, a.qr_ss, a.qr_sh, Hq, D, 1.f, stream);
      use_qrot(a);
    }
  }
  const dim3 grid((S + 127) / 128, Hq, B);
  // fa_fwd3: B1 S8192 Hq32 Hkv8 0.659 ms (834 TF/s; 977 TF/s at B4) vs 0.907 for the generic kernel;
  // RS = 2 (rmask): permlane32 row max, asm exp / row-sum pairs (2.091 -> 2.054 ms at B4 S8192); the widened
  // O store tail (T21) pays at short rows (B64 S512 0.343 -> 0.314 ms; profiles/r3_attention_wide_store_ab.jsonl)
  const unsigned nb1 = (unsigned)((S + 127) / 128 * Hq * B);
#define LLMT_FWD(DD)                                                  \
  if (!v3)                                                            \
    fa_fwd_kernel<DD><<<grid, 256, 0, stream>>>(a);                   \
  else if (a.rmask)                                                   \
    fa_fwd3_kernel<DD, 2, 1><<<nb1, 256, 0, stream>>>(a);             \
  else                                                                \
    fa_fwd3_kernel<DD, 1, 1, 4, true><<<nb1, 256, 0, stream>>>(a);
  switch (D) {
    case 64: { LLMT_FWD(64) } break;    // the v3 structure on 128-byte rows (256-byte LDS pitch)
    case 96: { LLMT_FWD(96) } break;    // Phi-3: 192-byte rows (256-byte LDS pitch)
    case 128: { LLMT_FWD(128) } break;
    default: return hipErrorInvalidValue;
  }
#undef LLMT_FWD
  return hipGetLastError();
}

// 1: a forward with fused RoPE needs no qrot scratch (the launch goes to fa_fwd3_kernel)
extern "C" int llmt_flash_attn_fwd_rope_inkernel(int D, float drop_p, int has_seg, int seg_runs) {
  (void)has_seg;
  (void)seg_runs;
  return fwd_uses_fwd3(D, drop_p > 0.f) ? 1 : 0;
}

// 1: the backward of this problem runs the generic kernels (GQA then needs the fp32 partials workspace)
extern "C" int llmt_flash_attn_bwd_generic(int D, float drop_p) {
  return (drop_p > 0.f || generic_only() || !(D == 64 || D == 96 || D == 128)) ? 1 : 0;
}

// floats of the `delta` workspace llmt_flash_attn_bwd needs
extern "C" int64_t llmt_flash_attn_bwd_ws(int B, int S, int Hq, int D) {
  const int64_t n = (int64_t)B * Hq * S;
  return (D == 128 || D == 96 || D == 64) ? n + (int64_t)B * Hq * ((S + 31) / 32) * kLdTile : n;
}

extern "C" hipError_t llmt_flash_attn_bwd(const void* q, const void* k, const void* v, const void* o,
                                          const void* dout, const float* lse, float* delta, const int* seg, void* dq,
                                          void* dk, void* dv, float* work, int B, int S, int Hq, int Hkv, int D,
                                          int64_t q_sb, int64_t q_ss, int64_t q_sh, int64_t k_sb, int64_t k_ss,
                                          int64_t k_sh, int64_t v_sb, int64_t v_ss, int64_t v_sh, int64_t o_sb,
                                          int64_t o_ss, int64_t o_sh, int64_t dq_sb, int64_t dq_ss, int64_t dq_sh,
                                          int64_t dk_sb, int64_t dk_ss, int64_t dk_sh, int64_t dv_sb, int64_t dv_ss,
                                          int64_t dv_sh, float scale, int causal, int window, int seg_runs,
                                          float drop_p, uint32_t drop_seed, const void* rpos, int rpos64,
                                          int64_t rp_sb, int64_t rp_ss, const float* rcos, const float* rsin,
                                          int64_t rP, void* qrot, float softcap, const float* slopes,
                                          const int* pend, void* olo, hipStream_t stream) {
  if (!(drop_p >= 0.f && drop_p < 1.f)) return hipErrorInvalidValue;
  if (!rope_ok(rpos, rcos, rsin, rP, rp_sb, rp_ss)) return hipErrorInvalidValue;
  // rope: dq / dk are returned for the unrotated q / k. qun: q holds UNROTATED queries (the forward rotated
  // them on load; qrot = scratch for the rotated rows); otherwise (qrot null) q / k are both rotated in
  // memory and only the inverse rotation of the gradients is fused
  const bool rope = rcos != nullptr, qun = rope && qrot != nullptr;
  if (Hkv <= 0 || Hq % Hkv) return hipErrorInvalidValue;
  if (!aligned16(q, q_sb, q_ss, q_sh) || !aligned16(k, k_sb, k_ss, k_sh) || !aligned16(v, v_sb, v_ss, v_sh) ||
      !aligned16(o, o_sb, o_ss, o_sh) || !aligned16(dout, o_sb, o_ss, o_sh) || !aligned16(dq, dq_sb, dq_ss, dq_sh) ||
      !aligned16(dk, dk_sb, dk_ss, dk_sh) || !aligned16(dv, dv_sb, dv_ss, dv_sh))
    return hipErrorInvalidValue;
  if (B == 0 || S == 0) return hipSuccess;
  if (!fits32(S, q_ss) || !fits32(S, k_ss) || !fits32(S, v_ss) || !fits32(S, o_ss)) return hipErrorInvalidValue;
  if (!strides32({q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh, dq_sb, dq_ss, dq_sh, dk_sb,
                  dk_ss, dk_sh, dv_sb, dv_ss, dv_sh}))
    return hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const bf16*)q; a.k = (const bf16*)k; a.v = (const bf16*)v; a.o = (const bf16*)o;
  a.dout = (const bf16*)dout; a.out = (bf16*)dq; a.lse = (float*)lse; a.delta = delta; a.seg = seg;
  if (seg && seg_runs) {
    a.rs = seg + (int64_t)B * S;
    a.re = seg + 2 * (int64_t)B * S;
    if (seg_runs == 2) {  // + the work orders of the query / key blocks
      a.qord = seg + 3 * (int64_t)B * S;
      a.kord = a.qord + (int64_t)B * ((S + 127) / 128);
    }
  }
  a.dk = (bf16*)dk; a.dv = (bf16*)dv;
  const int64_t part = (int64_t)B * S * Hq * D;
  a.dk_part = work; a.dv_part = work ? work + part : nullptr;
  a.B = B; a.S = S; a.Hq = Hq; a.Hkv = Hkv;
  a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh; a.k_sb = k_sb; a.k_ss = k_ss; a.k_sh = k_sh;
  a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh; a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
  a.d_sb = o_sb; a.d_ss = o_ss; a.d_sh = o_sh;  // dout shares O's layout (checked by the caller)
  a.dq_sb = dq_sb; a.dq_ss = dq_ss; a.dq_sh = dq_sh; a.dk_sb = dk_sb; a.dk_ss = dk_ss; a.dk_sh = dk_sh;
  a.dv_sb = dv_sb; a.dv_ss = dv_ss; a.dv_sh = dv_sh;
  a.scale = scale; a.causal = causal; a.window = window;
  set_dropout(a, drop_p, drop_seed);
  a.bmajor = bmajor_order();
  a.rmask = range_masks() && (seg == nullptr || a.rs != nullptr);
  a.early = early_dma();
  a.probe = attn_probe();
  const bool gqa = Hq != Hkv;
  const int64_t nrows = (int64_t)B * S * Hq;
  const dim3 grid((S + 127) / 128, Hq, B);
  const int dgrid = stream_grid(nrows, 256);
  // fused RoPE: with qun the dQ kernel rotates its rows on load and writes them to qrot for the dK/dV
  // kernel; the dQ / dK epilogues apply the inverse rotation. Generic kernels: qrot by the standalone
  // rotation, inverse passes after.
  if (rope) set_rope(a, rpos, rpos64, rp_sb, rp_ss, rcos, rsin, rP, qrot, D);
  if (!set_mod(a, softcap, slopes, pend, olo)) return hipErrorInvalidValue;
  if (const int mod = mod_of(a)) {
    if (!olo || !aligned16(olo, o_sb, o_ss, o_sh)) return hipErrorInvalidValue;
    a.ldw = delta + nrows;  // (as below)
    const hipError_t e = launch_mod_dq(a, D, mod, (unsigned)((S + 127) / 128 * Hq * B), stream);
    if (e != hipSuccess) return e;
    return launch_mod_dkdv(a, a.ldw, D, mod, (unsigned)((S + 127) / 128 * Hkv * B), stream);
  }
  if ((D == 128 || D == 96 || D == 64) && !a.drop_thresh && !generic_only()) {
    if (rope) {
      a.rope_q = qun;
      a.rope_dq = 1;
    }
    // delta buffer = [B, Hq, S] delta, then the packed per-tile row constants (llmt_flash_attn_bwd_ws),
    // written by the dQ kernel (its waves cover every 32-row tile of every head; the dK/dV kernel runs after
    // it on this stream)
    float* ld = delta + nrows;
    a.ldw = ld;
    const unsigned gq = (unsigned)((S + 127) / 128 * Hq * B), gk = (unsigned)((S + 127) / 128 * Hkv * B);
    // dK/dV ring: 8 slots for D = 128 (tiles 6 ahead; B4 S8192 backward 7.605 -> 7.544 ms in one process;
    // packed 32 docs/row 1.546 -> 1.511 ms), 6 for D = 96 / 64 (dense 3.635 vs 3.649 ms;
    // profiles/r5_dkdv_ring_ab.jsonl)
#define LLMT_BWD3(DD, RING)                                                       \
  if (a.rmask)                                                                    \
    fa_bwd_dq3_kernel<DD, true, true><<<gq, 256, 0, stream>>>(a);                 \
  else                                                                            \
    fa_bwd_dq3_kernel<DD, true, true, 4, true><<<gq, 256, 0, stream>>>(a);        \
  if (rope) {                                                                     \
    if (qun) use_qrot(a);                                                         \
    a.rope_q = a.rope_dq = 0;                                                     \
    a.rope_dk = 1;                                                                \
  }                                                                               \
  if (a.rmask)                                                                    \
    fa_bwd_dkdv5_kernel<DD, false, RING><<<gk, 256, 0, stream>>>(a, ld);          \
  else                                                                            \
    fa_bwd_dkdv5_kernel<DD, true><<<gk, 256, 0, stream>>>(a, ld);
    switch (D) {
      case 64: { LLMT_BWD3(64, 6) } break;
      case 96: { LLMT_BWD3(96, 6) } break;
      default: { LLMT_BWD3(128, 8) } break;
    }
#undef LLMT_BWD3
    return hipGetLastError();
  }
  if (gqa && !work) return hipErrorInvalidValue;
  if (qun) {  // the generic kernels: rotated queries in qrot, inverse passes over dq / dk below
    rope_launch(a, a.q, a.q_sb, a.q_ss, a.q_sh, a.qrot, a.qr_sb, a.qr_ss, a.qr_sh, Hq, D, 1.f, stream);
    use_qrot(a);
  }
#define LLMT_BWD(DD)                                                                              \
  fa_bwd_delta_kernel<DD><<<dgrid, 256, 0, stream>>>(a);                                          \
  fa_bwd_dq_kernel<DD><<<grid, 256, 0, stream>>>(a);                                              \
  if (gqa) {                                                                                      \
    fa_bwd_dkdv_kernel<DD, true><<<grid, 256, 0, stream>>>(a);                                    \
    fa_gqa_reduce_kernel<DD><<<stream_grid((int64_t)B * S * Hkv * (DD / 4), 256), 256, 0, stream>>>(a); \
  } else {                                                                                        \
    fa_bwd_dkdv_kernel<DD, false><<<grid, 256, 0, stream>>>(a);                                   \
  }
  switch (D) {
    case 64: { LLMT_BWD(64) } break;
    case 96: { LLMT_BWD(96) } break;
    case 128: { LLMT_BWD(128) } break;
    default: return hipErrorInvalidValue;
  }
#undef LLMT_BWD
  if (rope) {
    rope_launch(a, a.out, a.dq_sb, a.dq_ss, a.dq_sh, a.out, a.dq_sb, a.dq_ss, a.dq_sh, Hq, D, -1.f, stream);
    rope_launch(a, a.dk, a.dk_sb, a.dk_ss, a.dk_sh, a.dk, a.dk_sb, a.dk_ss, a.dk_sh, Hkv, D, -1.f, stream);
  }
  return hipGetLastError();
}
