// What each token sees (fh_attn_mask), and the entry points of attention under a mask.
#include "fh_masked.hpp"

namespace fh {
namespace {

constexpr int kMaskThreads = 256;

struct MaskDocs {
  const int64_t* starts;
  const int64_t* lengths;
  const int64_t* prefix;
  int64_t n;
  int seq_len;  // where starts is null
};

// Smallest of the values of 32 lanes.
__device__ __forceinline__ int min32(int v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, 32));
  return v;
}
__device__ __forceinline__ int max32(int v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 32));
  return v;
}

// One thread a token: its document by bisection, the ranges from the rule, their bounds
// over 32 tokens by exchanges.  Every end is clamped to the rows, so no value of the
// inputs can lead the attention kernels out of them.
__global__ __launch_bounds__(kMaskThreads) void k_attn_mask(MaskDocs docs, int T, int window, int causal,
                                                           int4* __restrict__ rows, int4* __restrict__ keys,
                                                           int4* __restrict__ queries) {
  const int t = static_cast<int>(blockIdx.x) * kMaskThreads + threadIdx.x;
  int begin = 0, end = 0;  // the token's document
  int64_t d = -1;
  if (t < T) {
    int64_t b, next;
    if (docs.starts != nullptr) {
      int64_t lo = 0, hi = docs.n;  // starts before lo are at or before t
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (docs.starts[mid] <= t) lo = mid + 1;
        else hi = mid;
      }
      d = lo - 1;
      b = d >= 0 ? docs.starts[d] : 0;
      next = lo < docs.n ? docs.starts[lo] : T;
    } else {
      d = t / docs.seq_len;
      b = d * docs.seq_len;
      next = b + docs.seq_len;
    }
    if (d >= 0) {
      b = max(b, int64_t{0});
      const int64_t room = max(min(next, static_cast<int64_t>(T)) - b, int64_t{0});
      const int64_t length = docs.lengths != nullptr ? min(max(docs.lengths[d], int64_t{0}), room) : room;
      if (t < b + length) {
        begin = static_cast<int>(b);
        end = static_cast<int>(b + length);
      }
    }
  }
  int4 r = make_int4(0, 0, 0, 0);
  if (begin < end) {
    const int first = window > 0 ? max(begin, t - window + 1) : begin;
    const int past = window > 0 ? static_cast<int>(min(static_cast<int64_t>(end), static_cast<int64_t>(t) + window)) : end;
    if (causal) {
      int prefix_end = begin;
      if (docs.prefix != nullptr)
        prefix_end = begin + static_cast<int>(min(max(docs.prefix[d], int64_t{0}), static_cast<int64_t>(end - begin)));
      r = make_int4(first, max(t + 1, prefix_end), t < prefix_end ? begin : t, past);
    } else {
      r = make_int4(first, past, first, past);
    }
  }
  if (t < T) rows[t] = r;
  const int tile = t / kMaskRows;
  const bool a = r.x < r.y, b = r.z < r.w;
  const int big = 0x7fffffff;
  const int4 kb = make_int4(min32(a ? r.x : big), max32(a ? r.y : 0), max32(a ? r.x : 0), min32(a ? r.y : big));
  const int4 qb = make_int4(min32(b ? r.z : big), max32(b ? r.w : 0), max32(b ? r.z : 0), min32(b ? r.w : big));
  if (t < T && t % kMaskRows == 0) {
    keys[tile] = kb;
    queries[tile] = qb;
  }
}

// Blocks of ROWS rows by falling length of what they look at, one workgroup for each of the
// table's orders: a counting sort in LDS.  (Blocks of one length come in any order, which no
// result depends on.)
__global__ __launch_bounds__(1024) void k_mask_order(MaskTable m, int T, int* __restrict__ order_q,
                                                     int* __restrict__ order_k128, int* __restrict__ order_k64) {
  __shared__ int at[1024];
  const int which = blockIdx.x, rows = which == 2 ? 64 : 128;
  const int4* bounds = which == 0 ? m.keys : m.queries;
  int* order = which == 0 ? order_q : which == 1 ? order_k128 : order_k64;
  const int n = (T + rows - 1) / rows, tiles = (T + kMaskRows - 1) / kMaskRows, per = rows / kMaskRows;
  const int unit = order_unit(T);
  auto bucket = [&](int i) {
    int lo = 0x7fffffff, hi = 0;
    for (int t = i * per; t < min((i + 1) * per, tiles); ++t) {
      lo = min(lo, bounds[t].x);
      hi = max(hi, bounds[t].y);
    }
    return hi > lo ? 1023 - min(1023, (hi - lo + unit - 1) / unit) : 1023;
  };
  const int tid = threadIdx.x;
  at[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) atomicAdd(&at[bucket(i)], 1);
  __syncthreads();
  const int mine = at[tid];
  for (int off = 1; off < 1024; off <<= 1) {
    const int add = tid >= off ? at[tid - off] : 0;
    __syncthreads();
    at[tid] += add;
    __syncthreads();
  }
  const int first = at[tid] - mine;
  __syncthreads();
  at[tid] = first;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) order[atomicAdd(&at[bucket(i)], 1)] = i;
}

constexpr float kMostScale = 1152921504606846976.f;  // what scores are made of stays finite
// tanh as 1 - 2 r is off by 2^-23 of the cap: from here on that would be more in a score than
// the rounding of a bf16 weight is in its logarithm (2^-9, halved twice).
constexpr float kMostCap = 4096.f;
// In fp32 scale / cap is a normal number, so that scores keep their bits, and cap * log2(e) finite.
constexpr float kMostCapF32 = 8.507059173023462e37f;  // 2^126
constexpr float kLeastRatioF32 = 1.1754943508222875e-38f;  // 2^-126

int check_tokens(const char* name, int64_t tokens) {
  if (tokens < 0 || tokens > (int64_t(1) << 30)) return fail(FH_ERR_INVALID, std::string(name) + ": tokens must be 0 to 2^30");
  return FH_OK;
}

}  // namespace

int masked_args(const char* name, fh_dtype dt, int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                float scale, float cap, const float* slopes, MaskedArgs& a) {
  const std::string n(name);
  if (dt != FH_BF16 && dt != FH_F32) return fail(FH_ERR_INVALID, n + ": dtype must be FH_BF16 or FH_F32");
  if (int e = check_tokens(name, tokens)) return e;
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65535)
    return fail(FH_ERR_INVALID, n + ": n_heads must be a positive multiple of n_kv_heads, at most 65535");
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return fail(FH_ERR_INVALID, n + ": head_dim must be 32, 64 or 128");
  if (!(scale > 0.f) || !(scale <= kMostScale)) return fail(FH_ERR_INVALID, n + ": scale must be positive, at most 2^60");
  if (!(cap >= 0.f) || !(cap < INFINITY)) return fail(FH_ERR_INVALID, n + ": cap must be 0 (none) or positive and finite");
  if (dt == FH_BF16 && cap > kMostCap) return fail(FH_ERR_INVALID, n + ": cap must be at most 4096 in bf16");
  if (dt == FH_F32 && cap > 0.f && !(cap <= kMostCapF32 && scale / cap >= kLeastRatioF32))
    return fail(FH_ERR_INVALID, n + ": cap must be at most 2^126, and 2^126 times the scale, in fp32");
  if (cap > 0.f && !(scale / cap <= kMostScale)) return fail(FH_ERR_INVALID, n + ": cap is too small for the scale");
  a.tokens = tokens;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.mode = (cap > 0.f ? kCap : 0) | (slopes != nullptr ? kBias : 0);
  const double log2e = 1.4426950408889634;
  a.score.scale = scale;
  a.score.scale_log2 = static_cast<float>(scale * log2e);
  a.score.in = cap > 0.f ? static_cast<float>(static_cast<double>(scale) / cap) : 0.f;
  a.score.in2 = cap > 0.f ? static_cast<float>(2.0 * log2e * scale / cap) : 0.f;
  a.score.cap_log2 = static_cast<float>(cap * log2e);
  a.score.slopes = slopes;
  return FH_OK;
}

int masked_stride(const char* name, const char* what, int64_t ld, int64_t heads, int64_t head_dim) {
  // < 2^24: the kernels' per-lane tile load offsets (up to 64 rows) are 32-bit
  if (ld < heads * head_dim || ld % 8 != 0 || ld >= (int64_t(1) << 24))
    return fail(FH_ERR_INVALID, std::string(name) + ": " + what +
                                    " row stride must be >= heads*head_dim, a multiple of 8 and < 2^24");
  return FH_OK;
}

}  // namespace fh

using namespace fh;

extern "C" int fh_packed_abi_version(void) { return FH_PACKED_ABI_VERSION; }

extern "C" size_t fh_attn_mask_size(int64_t tokens) {
  if (tokens <= 0 || tokens > (int64_t(1) << 30)) return 0;
  return mask_bytes(tokens);
}

extern "C" int fh_attn_mask(const int64_t* starts, const int64_t* lengths, const int64_t* prefix, int64_t n_documents,
                            int64_t tokens, int64_t seq_len, int64_t window, int causal, void* table,
                            hipStream_t stream) {
  if (int e = check_tokens("attn_mask", tokens)) return e;
  FH_REQUIRE(n_documents >= 0 && n_documents <= (int64_t(1) << 31), "attn_mask: bad number of documents");
  FH_REQUIRE(starts != nullptr || n_documents == 0 ||
                 (seq_len > 0 && seq_len <= tokens && tokens % seq_len == 0 && tokens / seq_len == n_documents),
             "attn_mask: without starts the documents' seq_len rows must make up the tokens");
  FH_REQUIRE(window >= 0, "attn_mask: window must be 0 (none) or positive");
  FH_REQUIRE(prefix == nullptr || (causal && window == 0), "attn_mask: a prefix goes with causal and without a window");
  if (tokens == 0) return FH_OK;
  FH_REQUIRE(table != nullptr && aligned16(table), "attn_mask: table must be 16-byte aligned");
  const MaskTable m = mask_table(table, tokens);
  if (n_documents == 0) starts = static_cast<const int64_t*>(table);  // none is read
  const int64_t most = int64_t(1) << 30;
  hipLaunchKernelGGL(k_attn_mask, dim3(static_cast<unsigned>((tokens + kMaskThreads - 1) / kMaskThreads)),
                     dim3(kMaskThreads), 0, stream,
                     MaskDocs{starts, lengths, prefix, n_documents, static_cast<int>(starts != nullptr ? 1 : seq_len)},
                     static_cast<int>(tokens), static_cast<int>(window < most ? window : most), causal ? 1 : 0,
                     const_cast<int4*>(m.rows), const_cast<int4*>(m.keys), const_cast<int4*>(m.queries));
  if (m.order_q != nullptr)
    hipLaunchKernelGGL(k_mask_order, dim3(3), dim3(1024), 0, stream, m, static_cast<int>(tokens),
                       const_cast<int*>(m.order_q), const_cast<int*>(m.order_k128), const_cast<int*>(m.order_k64));
  return check_launch("fh_attn_mask");
}

extern "C" int fh_masked_attn_fwd(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                  int64_t ldv, void* o, int64_t ldo, float* lse, int8_t* o_low, const void* table,
                                  int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, float scale, float cap,
                                  const float* slopes, hipStream_t stream) {
  const char* name = "masked_attn_fwd";
  MaskedArgs a;
  if (int e = masked_args(name, dt, tokens, n_heads, n_kv_heads, head_dim, scale, cap, slopes, a)) return e;
  if (int e = masked_stride(name, "q", ldq, n_heads, head_dim)) return e;
  if (int e = masked_stride(name, "k", ldk, n_kv_heads, head_dim)) return e;
  if (int e = masked_stride(name, "v", ldv, n_kv_heads, head_dim)) return e;
  if (int e = masked_stride(name, "o", ldo, n_heads, head_dim)) return e;
  if (tokens == 0) return FH_OK;
  FH_REQUIRE(q && k && v && o && table, "masked_attn_fwd: null pointer");
  FH_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(table),
             "masked_attn_fwd: pointers must be 16-byte aligned");
  FH_REQUIRE(o_low == nullptr || (dt == FH_BF16 && aligned16(o_low)),
             "masked_attn_fwd: o_low goes with bf16 and must be 16-byte aligned");
  const MaskedFwd c{q, k, v, ldq, ldk, ldv, o, ldo, lse, o_low, mask_table(table, tokens)};
  if (dt == FH_BF16) masked_fwd_bf16(c, a, stream);
  else masked_fwd_f32(c, a, stream);
  return check_launch("fh_masked_attn_fwd");
}

extern "C" size_t fh_masked_attn_bwd_workspace_size(fh_dtype dt, int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
                                                    int64_t head_dim) {
  MaskedArgs a;
  if (masked_args("masked_attn_bwd", dt, tokens, n_heads, n_kv_heads, head_dim, 1.f, 0.f, nullptr, a) || tokens == 0) return 0;
  return static_cast<size_t>(masked_workspace(dt, tokens, n_heads, n_kv_heads, head_dim).total) * sizeof(float);
}

extern "C" int fh_masked_attn_bwd(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                  int64_t ldv, const void* o, int64_t ldo, const void* dout, int64_t lddo,
                                  const float* lse, const int8_t* o_low, void* dq, int64_t lddq, void* dk, int64_t lddk, void* dv,
                                  int64_t lddv, const void* table, void* workspace, int64_t tokens, int64_t n_heads,
                                  int64_t n_kv_heads, int64_t head_dim, float scale, float cap, const float* slopes,
                                  hipStream_t stream) {
  const char* name = "masked_attn_bwd";
  MaskedArgs a;
  if (int e = masked_args(name, dt, tokens, n_heads, n_kv_heads, head_dim, scale, cap, slopes, a)) return e;
  struct Ld {
    int64_t ld, heads;
    const char* what;
  };
  const Ld lds[] = {{ldq, n_heads, "q"},       {ldk, n_kv_heads, "k"}, {ldv, n_kv_heads, "v"}, {ldo, n_heads, "o"},
                    {lddo, n_heads, "dout"},   {lddq, n_heads, "dq"},  {lddk, n_kv_heads, "dk"}, {lddv, n_kv_heads, "dv"}};
  for (const Ld& l : lds)
    if (int e = masked_stride(name, l.what, l.ld, l.heads, head_dim)) return e;
  if (tokens == 0) return FH_OK;
  FH_REQUIRE(q && k && v && o && dout && lse && dq && dk && dv && table && workspace, "masked_attn_bwd: null pointer");
  FH_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(dout) && aligned16(dq) &&
                 aligned16(dk) && aligned16(dv) && aligned16(table) && aligned16(workspace),
             "masked_attn_bwd: pointers must be 16-byte aligned");
  FH_REQUIRE((o_low != nullptr) == (dt == FH_BF16) && aligned16(o_low),
             "masked_attn_bwd: o_low goes with bf16 and must be 16-byte aligned");
  const MaskedBwd c{q,  k,    v,  o,    dout, ldq,  ldk, ldv, ldo, lddo, lse, o_low, dq, dk, dv, lddq, lddk, lddv,
                    mask_table(table, tokens), static_cast<float*>(workspace)};
  if (dt == FH_BF16) masked_bwd_bf16(c, a, stream);
  else masked_bwd_f32(c, a, stream);
  return check_launch("fh_masked_attn_bwd");
}
