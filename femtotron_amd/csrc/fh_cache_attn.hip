// Attention of a few new tokens of each sequence over a cache of its keys and values.
//
// Bound by the cache's bytes, each of which is read once: the query heads of a kv head and
// their new tokens are the columns of one product (32 a workgroup; more take several
// workgroups, which find the cache's rows in L2).
//
// Sequences are of lengths that only the device knows, so every workgroup works out its
// share by itself: the places that the sequences look at, one sequence after the other, are
// cut into `wanted` equal shares (a multiple of 128 places, at least 128), and workgroup i
// takes the i-th, be it a part of a sequence or several.  So one long sequence among short
// ones is spread over the chip like many equal ones, and a large room costs nothing.  What
// workgroup i sums of sequence b goes to slot i + b, which is no other's.
//
// A workgroup's waves take tiles of 32 places in turn, each for itself: its K and V go
// straight into the wave's own LDS, the next tile's while this one is multiplied, without a
// barrier (vmcnt alone).  S^T = K Q^T with one column a lane, an online softmax in fp32,
// O^T += V^T P^T, as in the forward under a mask; the waves' results meet in LDS, and the
// shares' in a second kernel.  Where the room is small or sequences are many, one workgroup
// takes a sequence, and there is no second kernel.
#include <algorithm>
#include <type_traits>

#include "fh_masked.hpp"

namespace fh {
namespace {

constexpr float kNoMax = -3.0e38f;  // finite: see the forward under a mask
constexpr int kPlaces = 32;         // of a tile
constexpr int kShare = 128;         // a share's places come in these

struct CacheArgs {
  const void *q, *k, *v;
  void* o;
  int64_t ldq, ldo, kb, kr, kh, vb, vr, vh;  // batch, row and head strides of k and v
  const int64_t* lengths;
  float* part;       // sums [item][HD * 32] (laid out by the kernels), or null: a workgroup a sequence
  float* stats;      // maximum and sum [item][2][32]
  int batch, n_new, room, nkv, group, window;
  int wanted;        // shares
  ScoreArgs score;
};

// The places [first, end) that sequence b's new tokens look at.
struct Span {
  int first, end;
};
__device__ __forceinline__ Span span_of(const CacheArgs& c, int b) {
  const int end = static_cast<int>(min(max(c.lengths[b], int64_t{0}), static_cast<int64_t>(c.room)));
  return {c.window > 0 ? max(0, end - c.n_new + 1 - c.window) : 0, end};
}

__device__ __forceinline__ int64_t wave_total(int64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// The lanes before this one, summed, and this one.
__device__ __forceinline__ int64_t wave_running(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int64_t up = __shfl_up(v, off, kWave);
    if (lane >= off) v += up;
  }
  return v;
}

// Places of a share, and of the sequences before `b` (all, b = batch): every wave of the chip
// works out the same.
struct Shares {
  int64_t share, before;
};
__device__ __forceinline__ Shares shares_of(const CacheArgs& c, int b, int lane) {
  int64_t all = 0, before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += kWave) {
    const int i = b0 + lane;
    if (i < c.batch) {
      const Span s = span_of(c, i);
      all += s.end - s.first;
      if (i < b) before += s.end - s.first;
    }
  }
  all = wave_total(all);
  const int64_t even = (all + c.wanted - 1) / c.wanted;
  return {max(int64_t{kShare}, (even + kShare - 1) / kShare * kShare), wave_total(before)};
}

// The sequence that holds place `at` of all of them, and the places before that sequence; b =
// batch: none does.
struct Found {
  int b;
  int64_t before;
};
__device__ __forceinline__ Found find(const CacheArgs& c, int64_t at, int lane) {
  int64_t before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += kWave) {
    const int i = b0 + lane;
    int64_t n = 0;
    if (i < c.batch) {
      const Span s = span_of(c, i);
      n = s.end - s.first;
    }
    const int64_t run = wave_running(n, lane);
    const uint64_t past = __ballot(before + run > at);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      return {b0 + l, before + __shfl(run - n, l, kWave)};
    }
    before += __shfl(run, kWave - 1, kWave);
  }
  return {c.batch, before};
}

// One tile of a wave: 32 places, of which the lane's column sees lo <= t < hi (less 4 hl).
template <int HD, int MODE, bool CAREFUL>
__device__ __forceinline__ void cache_tile(const char* K, const char* V, const bf16x8 (&qf)[HD / 16],
                                           f32x16 (&oacc)[HD / 32], float& m, float& l, int a_off, int b0, int b8,
                                           const float a, const float cap2, const float slope, float base, bool whole,
                                           int lo, int hi, int hl) {
  constexpr int NS = HD / 16, ND = HD / 32;
  f32x16 x = zero16();
#pragma unroll
  for (int s = 0; s < NS; ++s) x = mfma(lds_frag<HD>(K, a_off, 0, s), qf[s], x);
  float mloc = -INFINITY;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float z = x[j] * a;
    if constexpr (MODE & kCap) z = fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + fast_exp2(z)), cap2);
    if constexpr (MODE & kBias) z = fmaf(-slope, fabsf(base - acc_row(j, 0)), z);
    x[j] = z;
  }
  mask_range(x, !whole, !whole, lo, hi, 0, -INFINITY);
#pragma unroll
  for (int j = 0; j < 16; ++j) mloc = fmaxf(mloc, x[j]);
  mloc = xor32_max(mloc);
  if (wave_any(mloc > m + kRescaleSlack)) {
    const float mnew = fmaxf(m, mloc);
    const float alpha = fast_exp2(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) oacc[dt][j] *= alpha;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = fast_exp2(x[j] - m);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const bf16x8 pf = pack_frag(x, 8 * s);
    l = sum_bf16x8(pf, l);
    if constexpr (CAREFUL) {
      if (!whole) {
        wsum_careful<HD>(oacc, pf, V, b0, b8, 16 * s, lo + 4 * hl, hi + 4 * hl, hl);
        continue;
      }
    }
    wsum<HD>(oacc, pf, V, b0, b8, 16 * s);
  }
}

// The column of a lane: query head group_head of the kv head and new token u.
struct Column {
  int head, u;
  bool real;
};
__device__ __forceinline__ Column column_of(const CacheArgs& c, int kvh, int tile, int col) {
  const int i = tile * 32 + col, g = i / c.n_new;
  return {kvh * c.group + g, i - g * c.n_new, i < c.group * c.n_new};
}

// The part [begin, end) of sequence b's places for one kv head and column tile, to slot `slot`
// (or, without slots, to o).
template <int HD, int MODE, int WAVES>
__device__ __forceinline__ void cache_segment(const CacheArgs& c, char* lds, float (*sm)[32], float (*sl)[32], int b,
                                              int begin, int end, int seq_end, int slot) {
  constexpr int NS = HD / 16, ND = HD / 32, TILE = kPlaces * 2 * HD, RUNS = TILE / 1024, STEP = WAVES * kPlaces;
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.y, tile = blockIdx.z;
  const Column col = column_of(c, kvh, tile, l32);
  const int p = seq_end - c.n_new + col.u;  // the column's place
  // It sees places sees <= t < past of the part, which may be none where the sequence has some.
  const int sees = max(begin, c.window > 0 ? p + 1 - c.window : 0);
  const int past = col.real ? min(p + 1, end) : begin;
  const bool here = sees < past, some = col.real && p >= 0;
  // Every new token sees places [last_first, first_end).
  const int first_end = min(seq_end - c.n_new + 1, end), last_first = c.window > 0 ? max(0, seq_end - c.window) : 0;
  const float a = (MODE & kCap) ? c.score.in2 : c.score.scale_log2;
  const float slope = (MODE & kBias) && col.real ? c.score.slopes[col.head] * kLog2e : 0.f;

  const uint16_t* kp = static_cast<const uint16_t*>(c.k) + b * c.kb + kvh * c.kh;
  const uint16_t* vp = static_cast<const uint16_t*>(c.v) + b * c.vb + kvh * c.vh;
  TileDma<kPlaces, HD, 1> dk, dv;
  dk.init(c.kr, 0, lane);
  dv.init(c.vr, 0, lane);
  char* mine = lds + wave * 4 * TILE;
  const int from = begin + wave * kPlaces;
  const int n = from < end ? (end - from + STEP - 1) / STEP : 0;  // tiles
  auto load = [&](int i, char* st) __attribute__((always_inline)) {
    const int k0 = from + i * STEP;
    dk.load_asm(kp, c.kr, k0, seq_end - 1, st, 0, lane);
    dv.load_asm(vp, c.vr, k0, seq_end - 1, st + TILE, 0, lane);
  };
  bf16x8 qf[NS];
  {
    const uint16_t* row = static_cast<const uint16_t*>(c.q) + (static_cast<int64_t>(b) * c.n_new + col.u) * c.ldq +
                          static_cast<int64_t>(col.head) * HD + 8 * hl;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = col.real ? ld_frag(row + 16 * s) : as_bf16x8(make_uint4(0, 0, 0, 0));
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the loads below are counted from here
  int a_off = lane_off_a<HD>(lane);
  int b0 = lane_off_b<HD>(lane, 0), b8 = lane_off_b<HD>(lane, 8);
  f32x16 oacc[ND];
  float m, l;
  auto run = [&](auto careful) __attribute__((always_inline)) {
    m = kNoMax;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) oacc[dt] = zero16();
    if (n > 0) load(0, mine);
    for (int i = 0; i < n; ++i) {
      char* st = mine + (i & 1) * 2 * TILE;
      if (i + 1 < n) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other stage has been read
        load(i + 1, mine + ((i + 1) & 1) * 2 * TILE);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * RUNS) : "memory");
      } else {
        wait_loads();
      }
      refresh_offsets(a_off, b0, b8);
      const int k0 = from + i * STEP;
      const bool whole = k0 >= last_first && k0 + kPlaces <= first_end;
      cache_tile<HD, MODE, decltype(careful)::value>(st, st + TILE, qf, oacc, m, l, a_off, b0, b8, a, c.score.cap_log2,
                                                     slope, static_cast<float>(p - k0 - 4 * hl), whole,
                                                     sees - k0 - 4 * hl, past - k0 - 4 * hl, hl);
    }
  };
  run(std::false_type{});
  if (__builtin_expect(wave_any(here && not_finite<ND>(oacc)), 0)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    run(std::true_type{});
  }

  // The waves' results meet.
  const float lt = xor32_sum(l);
  if (hl == 0) {
    sm[wave][l32] = m;
    sl[wave][l32] = lt;
  }
  __syncthreads();  // also: every wave has read its tiles
  float mt = sm[0][l32];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) mt = fmaxf(mt, sm[w][l32]);
  const float alpha = fast_exp2(m - mt);
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += sl[w][l32] * fast_exp2(sm[w][l32] - mt);
  float(*red)[ND * 16][64] = reinterpret_cast<float(*)[ND * 16][64]>(lds);
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) red[wave][dt * 16 + j][lane] = here ? oacc[dt][j] * alpha : 0.f;  // (0 * inf is a NaN)
  __syncthreads();
  // The waves share the ND * 16 entries out, four dims at a time.
  const int64_t item = (static_cast<int64_t>(slot) * c.nkv + kvh) * gridDim.z + tile;
  if (c.part != nullptr && tid < 32) {
    c.stats[item * 64 + tid] = mt;
    c.stats[item * 64 + 32 + tid] = total;
  }
  for (int e = wave * 4; e < ND * 16; e += WAVES * 4) {  // entry dt * 16 + j
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = red[0][e + i][lane];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) x[i] += red[w][e + i][lane];
    }
    if (c.part != nullptr) {
      if (col.real) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c.part[item * (HD * 32) + (e + i) * 64 + lane] = x[i];
      }
    } else if (col.real) {
      const float mul = some ? 1.f / total : 0.f;
      uint16_t* row = static_cast<uint16_t*>(c.o) + (static_cast<int64_t>(b) * c.n_new + col.u) * c.ldo +
                      static_cast<int64_t>(col.head) * HD + (e >> 4) * 32 + acc_row(e & 15, hl);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = some ? x[i] * mul : 0.f;
      *reinterpret_cast<uint2*>(row) = make_uint2(pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3]));
    }
  }
}

// 32 sequences in a room of 8192, 32/8 heads of 128, capped: 100-105 us, 4.8-5.1 TB/s; 2 of up
// to 32768, 32 heads of 128, 5 new tokens: 135-141 us, 5.3-5.5; one of 2048, 32/4 heads of
// 64: 10 us, the loads of one workgroup a head one after another.
template <int HD, int MODE, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 1 : 2))) void k_cache_attn(CacheArgs c) {
  constexpr int TILE = kPlaces * 2 * HD;
  // [wave][stage][K, V]; the waves' sums meet in it afterwards.
  __shared__ __align__(16) char lds[WAVES * 4 * TILE];
  __shared__ float sm[WAVES][32], sl[WAVES][32];
  static_assert(HD / 32 * 16 * 64 * 4 <= 4 * TILE, "a wave's sums");
  const int lane = threadIdx.x & 63;
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  if (c.part == nullptr) {
    const int b = blockIdx.x;
    const Span s = span_of(c, b);
    cache_segment<HD, MODE, WAVES>(c, lds, sm, sl, b, uniform(s.first), uniform(s.end), uniform(s.end), 0);
    return;
  }
  const int64_t share = shares_of(c, 0, lane).share;
  int64_t at = share * blockIdx.x;
  const int64_t to = at + share;
  Found f = find(c, at, lane);
  for (int b = uniform(f.b); b < c.batch && at < to; ++b) {
    const Span s = span_of(c, b);
    const int64_t past = f.before + (s.end - s.first);  // the places up to this sequence's end
    if (past > at) {
      const int begin = s.first + static_cast<int>(max(at - f.before, int64_t{0}));
      const int end = s.first + static_cast<int>(min(to, past) - f.before);
      cache_segment<HD, MODE, WAVES>(c, lds, sm, sl, b, uniform(begin), uniform(end), uniform(s.end),
                                     static_cast<int>(blockIdx.x) + b);
      __syncthreads();  // the sums have been read
      at = min(to, past);
    }
    f.before = past;
  }
}

// One wave a query row: o = sum over its shares of 2^(m_s - M) sum_s / the same of the sums.
// What takes time is one load after another, so the sums are fetched eight at a time, before
// their weights are known.
template <typename T, int HD, int COLS>
__global__ __launch_bounds__(256) void k_cache_join(CacheArgs c) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = c.nkv * c.group;
  const int64_t rows = static_cast<int64_t>(c.batch) * c.n_new * heads;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (r >= rows) return;
  const int h = static_cast<int>(r % heads);
  const int64_t bu = r / heads;
  const int u = static_cast<int>(bu % c.n_new), b = static_cast<int>(bu / c.n_new);
  const Shares sh = shares_of(c, b, lane);
  const Span s = span_of(c, b);
  const int64_t len = s.end - s.first;
  const int first = static_cast<int>(sh.before / sh.share) + b;
  const int n = len > 0 ? static_cast<int>((sh.before + len - 1) / sh.share) + b - first + 1 : 0;
  const int kvh = h / c.group, i = (h - kvh * c.group) * c.n_new + u;
  const int tiles = (c.group * c.n_new + COLS - 1) / COLS, tile = i / COLS, col = i % COLS;
  const int64_t item0 = (static_cast<int64_t>(first) * c.nkv + kvh) * tiles + tile, step = static_cast<int64_t>(c.nkv) * tiles;
  constexpr int PER = (HD + 63) / 64;  // dims of a lane: lane + 64 i
  int64_t at[PER];
#pragma unroll
  for (int d = 0; d < PER; ++d) {
    const int dim = min(lane + 64 * d, HD - 1);
    if constexpr (COLS == 32) {  // [dim / 32][entry j][lane] of the accumulators
      const int in = dim & 31, hl = (in >> 2) & 1, j = ((in >> 3) << 2) + (in & 3);
      at[d] = (dim / 32 * 16 + j) * 64 + hl * 32 + col;
    } else {
      at[d] = col * HD + dim;
    }
  }
  float acc[PER], total = 0.f, m = kNoMax;
#pragma unroll
  for (int d = 0; d < PER; ++d) acc[d] = 0.f;
  for (int k0 = 0; k0 < n; k0 += kWave) {
    const int some = min(n - k0, kWave);
    float mk = kNoMax, lk = 0.f;
    if (lane < some) {
      const float* st = c.stats + (item0 + (k0 + lane) * step) * (2 * COLS) + col;
      mk = st[0];
      lk = st[COLS];
    }
    float v[8][PER];
    auto fetch = [&](int k) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < PER; ++d) v[e][d] = c.part[(item0 + (k0 + min(k + e, some - 1)) * step) * (HD * COLS) + at[d]];
    };
    fetch(0);
    const float mn = fmaxf(m, wave_max(mk)), alpha = fast_exp2(m - mn);
    m = mn;
    const float w = fast_exp2(mk - m);
    total = total * alpha + w * lk;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] *= alpha;
    for (int k = 0; k < some; k += 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float wk = __shfl(w, k + e, kWave);
#pragma unroll
        for (int d = 0; d < PER; ++d)
          if (k + e < some) acc[d] = fmaf(wk, v[e][d], acc[d]);
      }
      if (k + 8 < some) fetch(k + 8);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, kWave);
  const bool some = s.end - c.n_new + u >= 0;
  T* row = static_cast<T*>(c.o) + bu * c.ldo + static_cast<int64_t>(h) * HD;
#pragma unroll
  for (int d = 0; d < PER; ++d)
    if (lane + 64 * d < HD) Elem<T>::st1(row + lane + 64 * d, some ? acc[d] / total : 0.f);
}

// ------------------------------------------------------------------------ fp32
// The same on v_mfma_f32_16x16x4_f32, 16 columns a workgroup, operands straight from
// global memory (fp32 models: debugging and parity runs).
constexpr int kColsF32 = 16;

template <int HD, int MODE>
__device__ __forceinline__ void cache_segment_f32(const CacheArgs& c, float* tiles, float (*sm)[16], float (*sl)[16], int b,
                                                  int begin, int end, int seq_end, int slot) {
  constexpr int NU = HD / 16;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.y, tile = blockIdx.z;
  const int i = tile * kColsF32 + r, head = kvh * c.group + i / c.n_new, u = i % c.n_new;
  const bool real = i < c.group * c.n_new;
  const int p = seq_end - c.n_new + u;
  const int sees = real && c.window > 0 ? max(0, p + 1 - c.window) : 0, past = real ? min(p + 1, end) : 0;
  const bool some = real && p >= 0;
  const float a = (MODE & kCap) ? c.score.in : c.score.scale_log2;
  const float slope = (MODE & kBias) && real ? c.score.slopes[head] * kLog2e : 0.f;
  FragF32<HD> qf;
  if (real) {
    load_frag_f32<HD>(qf, static_cast<const float*>(c.q) + (static_cast<int64_t>(b) * c.n_new + u) * c.ldq +
                              static_cast<int64_t>(head) * HD, g);
  } else {
#pragma unroll
    for (int d = 0; d < NU; ++d) qf[d] = zero4();
  }
  f32x4 oacc[NU];
#pragma unroll
  for (int d = 0; d < NU; ++d) oacc[d] = zero4();
  float m = kNoMax, l = 0.f;
  const float* kp = static_cast<const float*>(c.k) + b * c.kb + kvh * c.kh;
  const float* vp = static_cast<const float*>(c.v) + b * c.vb + kvh * c.vh;
  for (int k0 = begin + 32 * wave; k0 < end; k0 += kShare) {
    const int lo = sees - k0, hi = past - k0;
    f32x4 x[2];
    float mloc = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      FragF32<HD> kf;
      load_frag_f32<HD>(kf, kp + static_cast<int64_t>(min(k0 + 16 * t + r, seq_end - 1)) * c.kr, g);
      x[t] = dot_f32<HD>(kf, qf);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 16 * t + 4 * g + e;
        float z = x[t][e] * a;
        if constexpr (MODE & kCap) z = tanhf(z) * c.score.cap_log2;
        if constexpr (MODE & kBias) z = fmaf(-slope, static_cast<float>(abs(p - k0 - n)), z);
        x[t][e] = n >= lo && n < hi ? z : -INFINITY;
        mloc = fmaxf(mloc, x[t][e]);
      }
    }
    const float mn = fmaxf(m, col_max(mloc));
    const float alpha = fast_exp2(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < NU; ++d) oacc[d] *= alpha;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = fast_exp2(x[t][e] - m);
        l += x[t][e];
      }
    wsum_f32<HD>(oacc, x, vp + static_cast<int64_t>(k0) * c.vr, c.vr, seq_end - 1 - k0, true, lo, hi, r, g);
  }
  l = col_sum(l);
  if (g == 0) {
    sm[wave][r] = m;
    sl[wave][r] = l;
  }
  __syncthreads();
  const float mt = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += sl[w][r] * fast_exp2(sm[w][r] - mt);
  const float mul = fast_exp2(m - mt) * (c.part != nullptr ? 1.f : 1.f / total);
#pragma unroll
  for (int d = 0; d < NU; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) oacc[d][e] = some ? oacc[d][e] * mul : 0.f;
  sum_waves_f32<HD, 4>(oacc, tiles, wave, r, g);
  if (wave == 0) put_tile_f32<HD>(tiles, oacc, r, g);
  __syncthreads();
  const int64_t item = (static_cast<int64_t>(slot) * c.nkv + kvh) * gridDim.z + tile;
  if (c.part != nullptr && threadIdx.x < 16) {
    c.stats[item * 32 + r] = mt;
    c.stats[item * 32 + 16 + r] = some ? total : 0.f;
  }
  for (int at = threadIdx.x; at < 16 * HD; at += 256) {
    const int row = at / HD, d = at % HD, j = tile * kColsF32 + row;
    if (j >= c.group * c.n_new) break;  // rows ascend with at
    const float x = tiles[row * (HD + 4) + d];
    if (c.part != nullptr) c.part[item * (HD * kColsF32) + at] = x;
    else
      static_cast<float*>(c.o)[(static_cast<int64_t>(b) * c.n_new + j % c.n_new) * c.ldo +
                               static_cast<int64_t>(kvh * c.group + j / c.n_new) * HD + d] = x;
  }
}

template <int HD, int MODE>
__global__ __launch_bounds__(256) void k_cache_attn_f32(CacheArgs c) {
  __shared__ __align__(16) float tiles[2 * 16 * (HD + 4)];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63;
  if (c.part == nullptr) {
    const Span s = span_of(c, blockIdx.x);
    cache_segment_f32<HD, MODE>(c, tiles, sm, sl, blockIdx.x, s.first, s.end, s.end, 0);
    return;
  }
  const int64_t share = shares_of(c, 0, lane).share;
  int64_t at = share * blockIdx.x;
  const int64_t to = at + share;
  Found f = find(c, at, lane);
  for (int b = f.b; b < c.batch && at < to; ++b) {
    const Span s = span_of(c, b);
    const int64_t past = f.before + (s.end - s.first);
    if (past > at) {
      cache_segment_f32<HD, MODE>(c, tiles, sm, sl, b, s.first + static_cast<int>(max(at - f.before, int64_t{0})),
                                  s.first + static_cast<int>(min(to, past) - f.before), s.end,
                                  static_cast<int>(blockIdx.x) + b);
      __syncthreads();
      at = min(to, past);
    }
    f.before = past;
  }
}

// ------------------------------------------------------------------------ host
// Workgroups that run at once: by their LDS one a CU at head_dim 128, two below.
int64_t workgroups(int64_t head_dim) { return head_dim == 128 ? 256 : 512; }

// Whether a workgroup takes a whole sequence: in small rooms, where the time is the loads one
// after another and the launches, and one more launch costs more than tiles in turn (bf16, calls
// of one sequence, in shares -> whole, 32/4 heads of 64: room 256 to 2048 18 -> 13 us, 4096 17.6
// -> 16.1, 8192 21 -> 28; 32/8 heads of 128: 1024 18 -> 13, 1536 17.3 -> 14.3, 2048 17.5 -> 17.3,
// 4096 22 -> 29; in fp32 up to 512 places at 64 and 256 at 128 18 -> 13, but 1024 at 64 18 -> 19
// and at 128 18 -> 34, 2048 at 64 18 -> 34); in larger ones where the sequences give workgroups enough by themselves, as shares of short sequences
// are several segments in turn and have to be joined.  The larger the room the more a single
// long sequence among short ones would cost, so there more workgroups are asked for.  bf16,
// lengths even over [1, room], in shares -> whole, 32/8 heads of 128: 64 sequences of 1280
// 47 -> 37 us, of 4096 132 -> 118, 128 of 8192 422 -> 399 (one long among short: 41 -> 23,
// 66 -> 41, 94 -> 87); 32/4 heads of 64: 256 of 8192 212 -> 199, but 128 of 16384 202 -> 225.
// The fp32 kernel takes a place slower: 256 of 8192 would go 355 -> 539.
bool whole_sequences(fh_dtype dt, int64_t room, int64_t head_dim, int64_t workgroups_of_all) {
  const int64_t small = head_dim == 128 ? 1024 : 2048;
  if (room <= small || dt == FH_F32) return room <= small;
  return (room <= 4 * small && workgroups_of_all >= workgroups(head_dim)) ||
         (room <= 8 * small && workgroups_of_all >= 2 * workgroups(head_dim));
}

struct CachePlan {
  int64_t tiles, wanted, slots, items;  // items: slots * kv heads * tiles
  bool split;
};

CachePlan cache_plan(fh_dtype dt, int64_t batch, int64_t n_new, int64_t room, int64_t n_heads, int64_t n_kv_heads,
                     int64_t head_dim) {
  CachePlan p{};
  const int64_t cols = dt == FH_BF16 ? 32 : kColsF32;
  p.tiles = (n_heads / n_kv_heads * n_new + cols - 1) / cols;
  p.split = !whole_sequences(dt, room, head_dim, batch * n_kv_heads * p.tiles);
  if (p.split) {
    p.wanted = std::max<int64_t>(1, workgroups(head_dim) / (n_kv_heads * p.tiles));
    p.wanted = std::min(p.wanted, batch * ((room + kShare - 1) / kShare));
    p.slots = p.wanted + batch;
  }
  p.items = p.slots * n_kv_heads * p.tiles;
  return p;
}

size_t stats_floats(const CachePlan& p, fh_dtype dt) { return static_cast<size_t>(p.items) * (dt == FH_BF16 ? 64 : 2 * kColsF32); }

int check_cache(fh_dtype dt, int64_t batch, int64_t n_new, int64_t room, int64_t n_heads, int64_t n_kv_heads,
                int64_t head_dim, float scale, float cap, const float* slopes, MaskedArgs& a) {
  if (int e = masked_args("cache_attn", dt, 0, n_heads, n_kv_heads, head_dim, scale, cap, slopes, a)) return e;
  FH_REQUIRE(batch >= 0 && n_new >= 0 && room >= 0, "cache_attn: negative sizes");
  FH_REQUIRE(room <= (int64_t(1) << 30) && batch <= (int64_t(1) << 20) && n_new <= (int64_t(1) << 20),
             "cache_attn: room must be at most 2^30, batch and n_new 2^20");
  FH_REQUIRE((n_heads / n_kv_heads * n_new + 15) / 16 <= 65535, "cache_attn: too many new tokens");
  FH_REQUIRE(batch * n_new * n_heads <= (int64_t(1) << 32), "cache_attn: too many rows");
  return FH_OK;
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" size_t fh_cache_attn_workspace_size(fh_dtype dt, int64_t batch, int64_t n_new, int64_t room, int64_t n_heads,
                                               int64_t n_kv_heads, int64_t head_dim) {
  MaskedArgs a;
  if (check_cache(dt, batch, n_new, room, n_heads, n_kv_heads, head_dim, 1.f, 0.f, nullptr, a) || batch == 0 ||
      n_new == 0 || room == 0)
    return 0;
  const CachePlan p = cache_plan(dt, batch, n_new, room, n_heads, n_kv_heads, head_dim);
  if (!p.split) return 0;
  const size_t cols = dt == FH_BF16 ? 32 : kColsF32;
  return (stats_floats(p, dt) + static_cast<size_t>(p.items) * cols * static_cast<size_t>(head_dim)) * sizeof(float);
}

extern "C" int fh_cache_attn(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t k_batch_stride,
                             int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_batch_stride,
                             int64_t v_row_stride, int64_t v_head_stride, void* o, int64_t ldo, const int64_t* lengths,
                             int64_t batch, int64_t n_new, int64_t room, int64_t n_heads, int64_t n_kv_heads,
                             int64_t head_dim, int64_t window, float scale, float cap, const float* slopes,
                             void* workspace, hipStream_t stream) {
  const char* name = "cache_attn";
  MaskedArgs a;
  if (int e = check_cache(dt, batch, n_new, room, n_heads, n_kv_heads, head_dim, scale, cap, slopes, a)) return e;
  FH_REQUIRE(window >= 0, "cache_attn: window must be 0 (none) or positive");
  if (batch == 0 || n_new == 0) return FH_OK;
  if (int e = masked_stride(name, "q", ldq, n_heads, head_dim)) return e;
  if (int e = masked_stride(name, "o", ldo, n_heads, head_dim)) return e;
  if (int e = masked_stride(name, "k", k_row_stride, 1, head_dim)) return e;
  if (int e = masked_stride(name, "v", v_row_stride, 1, head_dim)) return e;
  FH_REQUIRE(k_batch_stride % 8 == 0 && k_head_stride % 8 == 0 && v_batch_stride % 8 == 0 && v_head_stride % 8 == 0 &&
                 k_batch_stride >= 0 && k_head_stride >= 0 && v_batch_stride >= 0 && v_head_stride >= 0,
             "cache_attn: the cache's strides must be multiples of 8");
  FH_REQUIRE(q && o && lengths && (room == 0 || (k && v)), "cache_attn: null pointer");
  FH_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(workspace),
             "cache_attn: pointers must be 16-byte aligned");
  const CachePlan p = cache_plan(dt, batch, n_new, room, n_heads, n_kv_heads, head_dim);
  FH_REQUIRE(!p.split || workspace != nullptr, "cache_attn: null workspace");
  FH_REQUIRE(p.slots <= 0x7fffffff && n_kv_heads <= 65535, "cache_attn: grid too large");
  const int64_t most = int64_t(1) << 30;
  CacheArgs c{q, k, v, o, ldq, ldo, k_batch_stride, k_row_stride, k_head_stride, v_batch_stride, v_row_stride,
              v_head_stride, lengths, nullptr, nullptr, static_cast<int>(batch), static_cast<int>(n_new),
              static_cast<int>(room), static_cast<int>(n_kv_heads), static_cast<int>(n_heads / n_kv_heads),
              static_cast<int>(window < most ? window : most), static_cast<int>(p.wanted), a.score};
  if (p.split) {
    c.stats = static_cast<float*>(workspace);
    c.part = c.stats + stats_floats(p, dt);
  }
  const dim3 grid(static_cast<unsigned>(p.split ? p.wanted : batch), static_cast<unsigned>(n_kv_heads),
                  static_cast<unsigned>(p.tiles));
  const int64_t rows = batch * n_new * n_heads;
  const dim3 join(static_cast<unsigned>((rows + 3) / 4));
  dispatch_masked(head_dim, a.mode, [&](auto hd, auto mode) {
    constexpr int HD = decltype(hd)::value;
    constexpr int WHOLE = HD == 128 ? 4 : 8;  // waves of a workgroup that takes a sequence: 128 KB of LDS
    if (dt == FH_F32) hipLaunchKernelGGL((k_cache_attn_f32<HD, mode()>), grid, dim3(256), 0, stream, c);
    else if (p.split) hipLaunchKernelGGL((k_cache_attn<HD, mode(), 4>), grid, dim3(256), 0, stream, c);
    else hipLaunchKernelGGL((k_cache_attn<HD, mode(), WHOLE>), grid, dim3(64 * WHOLE), 0, stream, c);
    if (!p.split) return;
    if (dt == FH_BF16) hipLaunchKernelGGL((k_cache_join<uint16_t, HD, 32>), join, dim3(256), 0, stream, c);
    else hipLaunchKernelGGL((k_cache_join<float, HD, kColsF32>), join, dim3(256), 0, stream, c);
  });
  return check_launch("fh_cache_attn");
}
