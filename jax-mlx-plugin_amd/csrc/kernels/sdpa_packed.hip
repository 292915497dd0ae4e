// mfx_sdpa_packed, mfx_sdpa_packed_bwd: argument validation and kernel
// selection for attention over packed sequences.  The kernels are the packed
// instances of those of mfx_sdpa_fwd and mfx_sdpa_bwd (sdpa_packed.h): a
// workgroup finds its sequence on the device and then runs the same tiles.
//
// What bounds them is what bounds those: the matrix cores and the vector work
// between their products.  bf16, 32 heads on 8, D 128, causal: 16 sequences of 1
// .. 4096 tokens 330 - 365 us (0.83 - 0.92 PFLOP/s of visible pairs), 4095 + 12289
// 1.23 - 1.42 ms (1.1 to 0.97 PFLOP/s, by the clock); eight of 96 .. 2500 forward
// 146, dQ 207, dK / dV 357 us (in shares of the longest key blocks; whole 7% more).
//
// Roundings.  P, and in the backward dS, meet the matrix cores in the inputs'
// type, as in the unpacked kernels; sums, the softmax and delta are fp32.  Of
// the outputs' size (bf16, against 64 bits, their own rounding 0.0016): out off by
// 0.0020, dq and dk by 0.0025.  A second term of P or dS would cost another product
// beside the forward's two, or two beside the backward's seven.
#include <algorithm>
#include <cmath>

#include "sdpa_packed.h"

namespace mfx {
namespace {

enum class Kind { kNone, kFlash16, kFlashF32, kMfma16, kMfmaF32, kPadded16, kGeneric };

// Backward on the matrix cores: up to kPartBlocks blocks (four a CU) some are
// shared, at most kMaxParts ways (packed_share).
constexpr int kPartBlocks = 4 * kCus, kMaxParts = 8;

// Zeros in all of a [heads, T, D] tensor: a call without sequences.
template <typename T>
__global__ __launch_bounds__(256) void packed_zero_all(void* out, int64_t s1, int64_t s2, int64_t rows, int heads,
                                                       int D) {
  const int64_t st[4] = {0, s1, s2, 1};
  for (int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4)
    packed_zero_row<T>(out, st, (int)(r % heads), (int)(r / heads), D);
}

int zero_all(void* out, const int64_t* st, int64_t T, int64_t heads, int64_t D, int dtype, hipStream_t s) {
  if (!out) return fail(MFX_E_INVALID, "outputs must be non-null");
  if (st[2] != 1) return fail(MFX_E_INVALID, "feature (last) strides must be 1");
  const int64_t rows = T * heads;
  const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, 4096));
  if (dtype == MFX_F32)
    hipLaunchKernelGGL(packed_zero_all<float>, grid, dim3(256), 0, s, out, st[0], st[1], rows, (int)heads, (int)D);
  else  // (zero has the same bits in both 16-bit types)
    hipLaunchKernelGGL(packed_zero_all<bf16>, grid, dim3(256), 0, s, out, st[0], st[1], rows, (int)heads, (int)D);
  return launch_status("packed_zero_all");
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// (head, token, feature) strides as the kernels' (batch, head, seq, feature).
void bind(int64_t (&to)[4], const int64_t* st) {
  to[0] = 0;
  for (int i = 0; i < 3; ++i) to[i + 1] = st[i];
}

template <class Args>
int check_common(const Args* a) {
  if (a->T < 0 || a->num_seqs < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0)
    return fail(MFX_E_INVALID, "T and num_seqs must be >= 0, Hq, Hkv and D positive");
  if (a->Hq % a->Hkv != 0) return fail(MFX_E_INVALID, "Hq must be a multiple of Hkv");
  const int64_t lim = 0x7fffffffLL;
  if (a->T > lim || a->num_seqs >= lim || a->Hq > 65535 ||
      packed_slots(a->T, a->num_seqs, 32) * a->Hq > lim || a->T * a->Hq > lim)
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  if (a->dtype != MFX_F32 && a->dtype != MFX_BF16 && a->dtype != MFX_F16)
    return fail(MFX_E_UNSUPPORTED, "dtype must be f32, bf16 or f16");
  if (!std::isfinite(a->scale)) return fail(MFX_E_INVALID, "scale must be finite");
  if (a->D > 256) return fail(MFX_E_UNSUPPORTED, "head size above 256 is not supported");
  return MFX_OK;
}

// Whether the launches of a call fit: a wavefront a row, or workgroups of 256
// threads for blocks of 128 rows (the f32 ones of 64 threads for 32 rows have no
// more threads, and shares are only added to few blocks).
template <class Params>
int check_launch(const Params& p, Kind kind) {
  const int64_t rows = (int64_t)p.Hq * p.total;
  const bool fits = kind == Kind::kGeneric ? launch_fits((rows + 3) / 4, 256)
                                           : launch_fits(packed_slots(p.total, p.num_seqs, 128) * p.Hq, 256);
  return fits ? MFX_OK : fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
}

int plan_fwd(const mfx_sdpa_packed_args* a, SdpaParams& p, Kind& kind) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a)) return rc;
  kind = Kind::kNone;
  if (a->T == 0 || a->num_seqs == 0) return MFX_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->seq_offsets)
    return fail(MFX_E_INVALID, "q, k, v, out and seq_offsets must be non-null");
  for (const int64_t* st : {a->q_strides, a->k_strides, a->v_strides, a->o_strides})
    if (st[2] != 1) return fail(MFX_E_INVALID, "feature (last) strides must be 1");
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.lse = a->lse;
  bind(p.qs, a->q_strides);
  bind(p.ks, a->k_strides);
  bind(p.vs, a->v_strides);
  bind(p.os, a->o_strides);
  p.B = 1;
  p.Hq = (int)a->Hq;
  p.Hkv = (int)a->Hkv;
  p.Tq = p.Tk = p.total = (int)a->T;
  p.D = p.Dv = (int)a->D;
  p.group = (int)(a->Hq / a->Hkv);
  p.dtype = a->dtype;
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->scale * kLog2e;
  p.inv_scale_log2 = p.scale_log2 != 0.f ? 1.f / p.scale_log2 : 0.f;
  p.q_rms_eps = -1.f;
  p.num_splits = 1;
  p.split_len = p.Tk;
  p.seq_off = a->seq_offsets;
  p.num_seqs = (int)a->num_seqs;
  p.zero_rest = a->zero_rest;
  // (The 31-bit extents that the supports functions bound by Tk hold for every
  // sequence then; the row-block kernels of head size 256 are f32 only.)
  kind = p.D != 256 && flash_bf16_supports(p) ? Kind::kFlash16
         : flash_f32_supports(p)              ? Kind::kFlashF32
                                              : Kind::kGeneric;
  return check_launch(p, kind);
}

struct BwdPlan {
  SdpaBwdParams p{};
  Kind kind = Kind::kNone;
  size_t row_bytes = 0;            // delta
  size_t count_bytes = 0, sum_bytes = 0;  // blocks in shares: their counts and sums
  int dp = 0;                      // kPadded16: features of the padded copies
  size_t q_pad = 0, kv_pad = 0;    // bytes of one
};

// Shares of a head's `slots` blocks, `room` of which run at a time and which
// walk `tiles` more from one to the next: some while there are no more than
// kPartBlocks blocks, up to kMaxParts ways, and if any block can have them (their
// sums are two or more blocks a head: 268 MB for 100 tokens of 1024 heads).
void plan_shares(PackedShares& sh, int64_t slots, int heads, int room, int64_t tiles, size_t block_bytes, BwdPlan& pl) {
  const int64_t blocks = slots * heads;
  if (blocks > kPartBlocks) return;
  const int quarters = blocks <= 2 * kCus ? 3 : 4;
  if (!packed_shares_possible(pl.p.total, kBwdBlock, heads, quarters, room, tiles, kPartTiles)) return;
  sh.parts = (int)std::min<int64_t>(kMaxParts, kPartBlocks / blocks + 1);
  sh.quarters = quarters;
  // A block in k shares walks more than (k - 1) `most`, and all of a head
  // no more than `all`: so many blocks are shared at most, and so many
  // shares added.  (Of offsets that are no offsets there may be more
  // blocks than slots, but no workgroups behind slots + extra.)
  const int64_t all = room * 4 / sh.quarters / heads + 1;
  sh.extra = (int)std::min(slots * (sh.parts - 1), all);
  sh.shares = (int)std::min(slots, all) + sh.extra;
  const int64_t n = (int64_t)sh.shares * heads;
  pl.count_bytes += align256(n * sizeof(int));
  pl.sum_bytes += n * block_bytes;
}

int plan_bwd(const mfx_sdpa_packed_bwd_args* a, BwdPlan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a)) return rc;
  if (a->T == 0 || a->num_seqs == 0) return MFX_OK;
  if (!a->q || !a->k || !a->v || !a->dout || !a->out || !a->lse || !a->dq || !a->dk || !a->dv || !a->seq_offsets)
    return fail(MFX_E_INVALID, "q, k, v, dout, out, lse, dq, dk, dv and seq_offsets must be non-null");
  for (const int64_t* st : {a->q_strides, a->k_strides, a->v_strides, a->do_strides, a->o_strides, a->dq_strides,
                            a->dk_strides, a->dv_strides})
    if (st[2] != 1) return fail(MFX_E_INVALID, "feature (last) strides must be 1");
  SdpaBwdParams& p = pl.p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.dout = a->dout;
  p.o = a->out;
  p.lse = a->lse;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  bind(p.qs, a->q_strides);
  bind(p.ks, a->k_strides);
  bind(p.vs, a->v_strides);
  bind(p.dos, a->do_strides);
  bind(p.os, a->o_strides);
  bind(p.dqs, a->dq_strides);
  bind(p.dks, a->dk_strides);
  bind(p.dvs, a->dv_strides);
  p.B = 1;
  p.Hq = (int)a->Hq;
  p.Hkv = (int)a->Hkv;
  p.Tq = p.Tk = p.total = (int)a->T;
  p.D = p.Dv = (int)a->D;
  p.group = (int)(a->Hq / a->Hkv);
  p.dtype = a->dtype;
  p.causal = a->causal ? 1 : 0;
  p.scale = a->scale;
  p.scale_log2 = a->scale * kLog2e;
  p.seq_off = a->seq_offsets;
  p.num_seqs = (int)a->num_seqs;
  p.zero_rest = a->zero_rest;
  pl.row_bytes = align256((size_t)p.Hq * p.total * sizeof(float));
  pl.kind = Kind::kGeneric;
  if (bwd_mfma_supports(p)) {
    pl.kind = Kind::kMfma16;
  } else if (bwd_f32_supports(p)) {
    pl.kind = Kind::kMfmaF32;
  } else if ((p.dtype == MFX_BF16 || p.dtype == MFX_F16) && (p.D == 32 || p.D == 96)) {
    // On copies zero-padded to 64 / 128 features, as mfx_sdpa_bwd does: whole
    // 16-byte chunks, contiguous [heads][tokens][dp].
    bool chunked = true;
    for (const void* ptr : {p.q, p.k, p.v, p.dout, p.o, (const void*)p.dq, (const void*)p.dk, (const void*)p.dv})
      chunked = chunked && (uintptr_t)ptr % 16 == 0;
    for (const auto* st : {&p.qs, &p.ks, &p.vs, &p.dos, &p.os, &p.dqs, &p.dks, &p.dvs})
      for (int i = 1; i < 3; ++i) chunked = chunked && (*st)[i] % 8 == 0;
    SdpaBwdParams pp = p;
    const int dp = p.D == 32 ? 64 : 128;
    pp.D = pp.Dv = dp;
    for (auto* st : {&pp.qs, &pp.ks, &pp.vs, &pp.dos, &pp.os, &pp.dqs, &pp.dks, &pp.dvs}) {
      (*st)[1] = (int64_t)p.total * dp;
      (*st)[2] = dp;
    }
    pp.q = pp.k = pp.v = pp.dout = pp.o = nullptr;
    pp.dq = pp.dk = pp.dv = nullptr;
    if (chunked && bwd_mfma_supports(pp)) {
      pl.kind = Kind::kPadded16;
      pl.dp = dp;
      pl.q_pad = align256((size_t)p.Hq * p.total * dp * 2);
      pl.kv_pad = align256((size_t)p.Hkv * p.total * dp * 2);
    }
  }
  if (int rc = check_launch(p, pl.kind)) return rc;
  if ((pl.kind == Kind::kMfma16 || pl.kind == Kind::kPadded16) && p.causal && p.num_seqs <= 64 * kLaneSeqs) {
    // dK, dV: a key block walks all queries behind it for every head of its group, and
    // the longest ones alone can last longer than a CU's part of the whole
    // (backward of one sequence of 4096 tokens, 32 heads on 8: 730 us with whole
    // blocks, 602 with shares of at most three quarters of that part, 646 of
    // one; 512 tokens: 100 and 59; 3000 tokens in 2, 8 heads on 1: 580 and 144).
    // With more than two blocks a CU smaller ones fill the gaps and joining
    // shares costs more (8192 tokens in 1: 1990 whole, 2055 in three quarters;
    // in 8 of 96 .. 2500: 622, 614, and 607 in shares of one part).
    const int64_t slots = packed_slots(p.total, p.num_seqs, kBwdBlock);
    const size_t block_bytes = (size_t)kBwdBlock * (pl.dp ? pl.dp : p.D) * sizeof(float);
    plan_shares(p.key_shares, slots, p.Hkv, kCus, 2 * (int64_t)p.group, 2 * block_bytes, pl);
    // dQ: blocks of queries, of which two run on a CU; counts that nothing before
    // it clears cost a launch, 2 to 4 us.  (Whole backward, shares of queries and
    // none: 8192 tokens, 4 heads on 1, 457 and 524 us; 12289 in 2 heads, 420 and
    // 564; 1500 + 700, 4 heads, 86 and 100.  But 8192, 8 on 2, 698 and 686; four
    // of 512, 8 heads, 55 and 51.)
    if (p.total > 2048 && slots * p.Hq <= 2 * kCus)
      plan_shares(p.query_shares, slots, p.Hq, 2 * kCus, 2, block_bytes, pl);
  }
  return MFX_OK;
}

size_t bwd_bytes(const BwdPlan& pl) {
  return pl.kind == Kind::kNone
             ? 0
             : pl.row_bytes + pl.count_bytes + pl.sum_bytes + (pl.dp ? 4 * pl.q_pad + 4 * pl.kv_pad : 0);
}

int run_padded(const BwdPlan& pl, char* w, hipStream_t s) {
  const SdpaBwdParams& p = pl.p;
  SdpaBwdParams pp = p;
  pp.zero_rest = 0;  // (the copies' rows in no sequence reach no output)
  pp.D = pp.Dv = pl.dp;
  for (auto* st : {&pp.qs, &pp.ks, &pp.vs, &pp.dos, &pp.os, &pp.dqs, &pp.dks, &pp.dvs}) {
    (*st)[1] = (int64_t)p.total * pl.dp;
    (*st)[2] = pl.dp;
  }
  char* wk = w + 4 * pl.q_pad;
  struct Copy {
    const void* src;
    void* dst;
    int H;
    const int64_t* st;
    bool zero;
  };
  const Copy in[5] = {{p.q, w, p.Hq, p.qs},
                      {p.dout, w + pl.q_pad, p.Hq, p.dos},
                      {p.o, w + 2 * pl.q_pad, p.Hq, p.os},
                      {p.k, wk, p.Hkv, p.ks},
                      {p.v, wk + pl.kv_pad, p.Hkv, p.vs}};
  for (const Copy& c : in)
    if (int rc = packed_pad_rows(c.src, c.dst, p, c.H, pl.dp, c.st, false, false, s)) return rc;
  pp.q = in[0].dst;
  pp.dout = in[1].dst;
  pp.o = in[2].dst;
  pp.k = in[3].dst;
  pp.v = in[4].dst;
  pp.dq = w + 3 * pl.q_pad;
  pp.dk = wk + 2 * pl.kv_pad;
  pp.dv = wk + 3 * pl.kv_pad;
  if (int rc = launch_packed_bwd_mfma(pp, s)) return rc;
  const Copy out[3] = {{pp.dq, p.dq, p.Hq, p.dqs, (p.zero_rest & 1) != 0},
                       {pp.dk, p.dk, p.Hkv, p.dks, (p.zero_rest & 2) != 0},
                       {pp.dv, p.dv, p.Hkv, p.dvs, (p.zero_rest & 4) != 0}};
  for (const Copy& c : out)
    if (int rc = packed_pad_rows(c.src, c.dst, p, c.H, pl.dp, c.st, true, c.zero, s)) return rc;
  return MFX_OK;
}

const char* name_of(Kind kind, int dtype, int D) {
  static const char* const f16[2][4] = {
      {"packed_bf16_d32", "packed_bf16_d64", "packed_bf16_d96", "packed_bf16_d128"},
      {"packed_f16_d32", "packed_f16_d64", "packed_f16_d96", "packed_f16_d128"}};
  static const char* const f32[5] = {"packed_f32_d32", "packed_f32_d64", "packed_f32_d96", "packed_f32_d128",
                                     "packed_f32_d256"};
  switch (kind) {
    case Kind::kNone: return "none";
    case Kind::kGeneric: return "packed_generic";
    case Kind::kFlashF32:
    case Kind::kMfmaF32: return f32[D == 256 ? 4 : D / 32 - 1];
    default: return f16[dtype == MFX_F16][D / 32 - 1];
  }
}

}  // namespace
}  // namespace mfx

extern "C" {

const char* mfx_sdpa_packed_kernel_name(const mfx_sdpa_packed_args* args) {
  mfx::SdpaParams p{};
  mfx::Kind kind;
  if (mfx::plan_fwd(args, p, kind) != MFX_OK) return nullptr;
  return mfx::name_of(kind, args->dtype, (int)args->D);
}

int mfx_sdpa_packed(const mfx_sdpa_packed_args* args, void* stream) {
  using namespace mfx;
  SdpaParams p{};
  Kind kind;
  if (int rc = plan_fwd(args, p, kind)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (kind) {
    case Kind::kNone:
      if (args->T == 0 || !args->zero_rest) return MFX_OK;
      return zero_all(args->out, args->o_strides, args->T, args->Hq, args->D, args->dtype, s);
    case Kind::kFlash16: return launch_packed_flash16(p, s);
    case Kind::kFlashF32: return launch_packed_f32(p, s);
    default: return launch_packed_generic(p, s);
  }
}

const char* mfx_sdpa_packed_bwd_kernel_name(const mfx_sdpa_packed_bwd_args* args) {
  mfx::BwdPlan pl;
  if (mfx::plan_bwd(args, pl) != MFX_OK) return nullptr;
  return mfx::name_of(pl.kind, args->dtype, (int)args->D);
}

size_t mfx_sdpa_packed_bwd_workspace_size(const mfx_sdpa_packed_bwd_args* args) {
  mfx::BwdPlan pl;
  if (mfx::plan_bwd(args, pl) != MFX_OK) return 0;
  return mfx::bwd_bytes(pl);
}

int mfx_sdpa_packed_bwd(const mfx_sdpa_packed_bwd_args* args, void* stream) {
  using namespace mfx;
  BwdPlan pl;
  if (int rc = plan_bwd(args, pl)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (pl.kind == Kind::kNone) {
    struct Out {
      void* p;
      const int64_t* st;
      int64_t heads;
    };
    const Out outs[3] = {{args->dq, args->dq_strides, args->Hq},
                         {args->dk, args->dk_strides, args->Hkv},
                         {args->dv, args->dv_strides, args->Hkv}};
    for (int i = 0; i < 3; ++i)
      if (args->T > 0 && (args->zero_rest >> i & 1))
        if (int rc = zero_all(outs[i].p, outs[i].st, args->T, outs[i].heads, args->D, args->dtype, s)) return rc;
    return MFX_OK;
  }
  const size_t need = bwd_bytes(pl);
  char* ws = nullptr;
  if (args->workspace) {
    if (args->workspace_bytes < need)
      return fail(MFX_E_WORKSPACE, "workspace smaller than mfx_sdpa_packed_bwd_workspace_size()");
    if ((uintptr_t)args->workspace % 256) return fail(MFX_E_INVALID, "workspace must be 256-byte aligned");
    ws = static_cast<char*>(args->workspace);
  } else {
    ws = static_cast<char*>(device_scratch(need, s));
    if (!ws) return MFX_E_HIP;
  }
  pl.p.delta = reinterpret_cast<float*>(ws);
  ws += pl.row_bytes;
  for (PackedShares* sh : {&pl.p.key_shares, &pl.p.query_shares}) {
    const size_t n = (size_t)sh->shares * (sh == &pl.p.key_shares ? pl.p.Hkv : pl.p.Hq);
    sh->count = reinterpret_cast<int*>(ws);
    ws += align256(n * sizeof(int));
    sh->sums = reinterpret_cast<float*>(ws);
    ws += n * kBwdBlock * (pl.dp ? pl.dp : pl.p.D) * (sh == &pl.p.key_shares ? 2 : 1) * sizeof(float);
  }
  switch (pl.kind) {
    case Kind::kMfma16: return launch_packed_bwd_mfma(pl.p, s);
    case Kind::kMfmaF32: return launch_packed_bwd_f32(pl.p, s);
    case Kind::kPadded16: return run_padded(pl, ws, s);
    default: return launch_packed_bwd_generic(pl.p, s);
  }
}

}  // extern "C"
