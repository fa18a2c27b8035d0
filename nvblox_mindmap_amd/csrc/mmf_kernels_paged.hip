// mmf_kernels_paged.hip -- the paged context memory of the policy's attention: keys and values of growing contexts in pages of P tokens,
// appended with the position rotation on the way, read by the attention of a few new tokens, and by the attention over the pages that a
// cheap score selects.
//
//   keys   [num_pages, H, P, W]   a token's channels side by side   (W: the head size rounded up; channels >= head_dim are zero)
//   values [num_pages, H, W, P]   a channel's tokens side by side
//   key_min, key_max [num_pages, H, W]   smallest / largest stored key of the page per channel
//   table  [B, slots] int32       page of a context's tokens slot * P .. slot * P + P - 1; an entry outside [0, num_pages) holds nothing
//
// Every address below is a page in [0, num_pages) and a slot in [0, P): entries that the device data make invalid are replaced by page 0
// and masked, so no table, length or offset can lead a read or write out of the pools.
#include <float.h>

#include <algorithm>
#include <cmath>

#include "mmf_device.h"
#include "mmf_launch_policy.h"

namespace mmf {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));

template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <class T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}

// a computed value in its storage type: one value for every use of it (without the barrier the compiler may convert inside the last
// multiplication for one use and after it for another)
template <class T>
__device__ __forceinline__ T stored(float x) {
  asm("" : "+v"(x));
  return (T)x;
}

// the smaller / larger of two; NaN if either is (a page that holds a NaN key shows it)
__device__ __forceinline__ float smaller(float a, float b) { return (b < a || b != b) ? b : a; }
__device__ __forceinline__ float larger(float a, float b) { return (b > a || b != b) ? b : a; }

// ---- append ---------------------------------------------------------------------------------------------------------------------------
// Token i of the rows offsets[b] .. offsets[b + 1] - 1 becomes token starts[b] + i - offsets[b] of context b.  A workgroup owns one
// (context, page) pair and a range of heads, so a page's summary has one writer and needs no atomics; it finds its pair by a scan over
// the contexts' page counts.  A thread takes VEC channels of VT neighbouring slots: the keys go out row by row as they came, the values
// are transposed in its registers so that both stores are wide.
struct AppendArgs {
  const void *k, *v;
  long long k_stride, v_stride;
  const float* positions;
  int axes, rotary;   // rotary channels: of every head (rotary <= hd) or of the whole row
  double log2_base;
  const int *offsets, *starts, *table;
  int B, slots, n_tokens, pshift, H, hd, W, num_pages, heads_per_wg;
  void *keys, *values, *kmin, *kmax;
};

struct Segment {
  int b, slot, first, last, row;  // context, table slot, slots [first, last) of the page, row of slot `first`'s token
};

// The unit-th (context, page) pair that gets tokens: contexts in order, pages in order.
__device__ __forceinline__ bool find_segment(const AppendArgs& a, int unit, Segment& s) {
  const int lane = threadIdx.x & 63, P = 1 << a.pshift;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int lo = 0, n = 0, st = 0, np = 0;
    if (b < a.B) {
      lo = min(max(a.offsets[b], 0), a.n_tokens);
      const int hi = min(max(a.offsets[b + 1], 0), a.n_tokens);
      st = a.starts[b];
      n = st >= 0 ? max(hi - lo, 0) : 0;
      // (tokens behind the table's last slot have no page)
      const long long room = (long long)a.slots * P - st;
      n = room <= 0 ? 0 : (int)min((long long)n, room);
      np = n > 0 ? ((st + n - 1) >> a.pshift) - (st >> a.pshift) + 1 : 0;
    }
    int upto = np;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    const unsigned long long hit = __ballot(before + upto > unit);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      const int base = before + __shfl(upto, src) - __shfl(np, src);
      const int st_ = __shfl(st, src), n_ = __shfl(n, src), lo_ = __shfl(lo, src);
      s.b = b0 + src;
      s.slot = (st_ >> a.pshift) + unit - base;
      const int page_first = s.slot << a.pshift;
      s.first = max(st_ - page_first, 0);
      s.last = min(st_ + n_ - page_first, P);
      s.row = lo_ + page_first + s.first - st_;
      return true;
    }
    before += __shfl(upto, 63);
  }
  return false;
}

// cos / sin of the angle of channel pair `within` / 2 at a position: position * base^(-2 j / span), taken in turns and reduced in 64
// bits (a far position times a frequency loses its fraction in 32), then in 32 bits on [-1/2, 1/2] turns.
__device__ __forceinline__ double turns_per_unit(int within, int span, double log2_base) {
  const int j2 = (within % span) & ~1;
  return exp2(-log2_base * (double)j2 / (double)span) * 0.15915494309189533576888;
}
__device__ __forceinline__ void turn(float position, double freq, float& c, float& s) {
  const double t = (double)position * freq;
  sincospif(2.0f * (float)(t - rint(t)), &s, &c);
}

template <class TI, class T, int VEC, int VT>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  Segment seg;
  if (!find_segment(a, blockIdx.x, seg)) return;
  const int page = a.table[(long long)seg.b * a.slots + seg.slot];
  if (page < 0 || page >= a.num_pages) return;
  const int h0 = blockIdx.y * a.heads_per_wg, nh = min(a.heads_per_wg, a.H - h0);
  const int chunks_per_head = a.hd / VEC, nchunks = nh * chunks_per_head;
  const int g0 = seg.first / VT, ng = (seg.last - 1) / VT + 1 - g0;
  int gw = 1;  // neighbouring lanes take neighbouring slot groups: 8 of them fill the value rows' cache lines
  while (gw < 8 && gw < ng) gw <<= 1;
  const int gl = threadIdx.x & (gw - 1);
  const TI* __restrict__ kin = (const TI*)a.k;
  const TI* __restrict__ vin = (const TI*)a.v;
  const long long page_head = (long long)page * a.H;
  for (int ch = threadIdx.x / gw; ch < nchunks; ch += 256 / gw) {
    const int h = h0 + ch / chunks_per_head, d = (ch % chunks_per_head) * VEC;
    const int c = h * a.hd + d;  // channel in the row
    const int within = a.rotary > a.hd ? c : d;
    const int span = a.rotary ? a.rotary / a.axes : 1;
    T* __restrict__ kp = (T*)a.keys + ((page_head + h) << a.pshift) * a.W + d;
    T* __restrict__ vp = (T*)a.values + (((page_head + h) * a.W + d) << a.pshift);
    // VEC > 1: the pairs are the lane's own; VEC == 1: the partner is the neighbouring channel
    constexpr int NPAIR = VEC > 1 ? VEC / 2 : 1;
    double freq[NPAIR];
    int axis[NPAIR];
#pragma unroll
    for (int i = 0; i < NPAIR; ++i) {
      const int w = within + 2 * i;
      const bool on = w < a.rotary;
      axis[i] = on ? w / span : -1;
      freq[i] = on ? turns_per_unit(w, span, a.log2_base) : 0.0;
    }
    float lo[VEC], hi[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      lo[i] = INFINITY;
      hi[i] = -INFINITY;
    }
    for (int g = gl; g < ng; g += gw) {
      const int slot0 = (g0 + g) * VT;
      T vt[VEC][VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        const int slot = slot0 + t;
        const bool in = slot >= seg.first && slot < seg.last;
        if (!in) continue;
        const long long row = seg.row + (slot - seg.first);
        float x[VEC];
        const TI* kr = kin + row * a.k_stride + c;
        const TI* vr = vin + row * a.v_stride + c;
        if constexpr (VEC > 1) {
          const Pack<TI, VEC> kv = *reinterpret_cast<const Pack<TI, VEC>*>(kr);
          const Pack<TI, VEC> vv = *reinterpret_cast<const Pack<TI, VEC>*>(vr);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            x[i] = to_f(kv.v[i]);
            vt[i][t] = (T)to_f(vv.v[i]);
          }
          if (a.rotary) {
#pragma unroll
            for (int i = 0; i < NPAIR; ++i)
              if (axis[i] >= 0) {
                float cs, sn;
                turn(a.positions[row * a.axes + axis[i]], freq[i], cs, sn);
                const float e = x[2 * i], o = x[2 * i + 1];
                x[2 * i] = e * cs - o * sn;
                x[2 * i + 1] = o * cs + e * sn;
              }
          }
        } else {
          x[0] = to_f(kr[0]);
          vt[0][t] = (T)to_f(vr[0]);
          if (axis[0] >= 0) {
            float cs, sn;
            turn(a.positions[row * a.axes + axis[0]], freq[0], cs, sn);
            const bool odd = within & 1;
            const float p = to_f(kr[odd ? -1 : 1]);
            x[0] = odd ? x[0] * cs + p * sn : x[0] * cs - p * sn;
          }
        }
        Pack<T, VEC> out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          out.v[i] = stored<T>(x[i]);  // the one rounding of a key; the summary is of the stored value
          const float y = to_f(out.v[i]);
          lo[i] = smaller(lo[i], y);
          hi[i] = larger(hi[i], y);
        }
        if constexpr (VEC > 1)
          *reinterpret_cast<Pack<T, VEC>*>(kp + (long long)slot * a.W) = out;
        else
          kp[(long long)slot * a.W] = out.v[0];
      }
      if (slot0 >= seg.first && slot0 + VT <= seg.last) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          Pack<T, VT> out;
#pragma unroll
          for (int t = 0; t < VT; ++t) out.v[t] = vt[i][t];
          *reinterpret_cast<Pack<T, VT>*>(vp + ((long long)i << a.pshift) + slot0) = out;
        }
      } else {
#pragma unroll
        for (int t = 0; t < VT; ++t)
          if (slot0 + t >= seg.first && slot0 + t < seg.last) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) vp[((long long)i << a.pshift) + slot0 + t] = vt[i][t];
          }
      }
    }
    // over the gw lanes of this chunk, then with what the page held before (a page's summary begins with its first slot)
    T* __restrict__ mn = (T*)a.kmin + (page_head + h) * a.W + d;
    T* __restrict__ mx = (T*)a.kmax + (page_head + h) * a.W + d;
    const bool merge = seg.first > 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float l = lo[i], u = hi[i];
      for (int m = 1; m < gw; m <<= 1) {
        l = smaller(l, __shfl_xor(l, m));
        u = larger(u, __shfl_xor(u, m));
      }
      if (gl == 0) {
        if (merge) {
          l = smaller(l, to_f(mn[i]));
          u = larger(u, to_f(mx[i]));
        }
        mn[i] = (T)l;
        mx[i] = (T)u;
      }
    }
  }
}

// ---- attention over pages ---------------------------------------------------------------------------------------------------------------
// softmax(q k^T scale) v of the query rows that share a key-value head, over virtual keys i = entry * P + offset: entry e is table slot
// e, or slot selected[e].  A workgroup of 4 waves takes a run of keys of one unit (context, key-value head, 16 RT rows); the waves take
// tiles of 32 keys in turn, each with a running maximum and sum of its own, merged through LDS at the end.  Both products run on the
// matrix cores without a pass through LDS: S^T = K Q^T leaves lane group g of a tile with the scores of its keys, which are the operand
// that O^T = V^T P^T takes from that lane group -- the rows of K are dealt out so that they are 8 neighbouring keys (4 in 32-bit pages), i.e. one
// 16-byte load of a value row.  What bounds it is the single pass over keys and values.
struct AttArgs {
  const void *q, *keys, *values;
  const int *table, *lengths, *selected;
  int B, T, heads, H, G, hd, slots, num_pages, pshift, count;  // G = heads / H; count: entries of `selected` per (b, t, head)
  int rows, row_blocks, splits;                               // rows of a unit
  float scale_log2;
  void* out;
  float* part;  // [unit, split, 16 RT, W] then [unit, split, 16 RT, 2]
};

template <class T>
struct Mma;
template <>
struct Mma<_Float16> {
  using V8 = h8v;
  static __device__ __forceinline__ f32x4 k32(h8v x, h8v y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 k16(uint2 x, uint2 y, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4v, x), __builtin_bit_cast(h4v, y), c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  using V8 = b8v;
  static __device__ __forceinline__ f32x4 k32(b8v x, b8v y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 k16(uint2 x, uint2 y, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4v, x), __builtin_bit_cast(s4v, y), c, 0, 0, 0);
  }
};

// Weights of 16-bit pages are exp2(s - m + kLift): half's smallest step is then 2^-31 of the largest weight (bfloat16 and float32 have
// the exponents), and the largest, 2^(8 + kLift), still fits.  The factor is in the weights and in their sum alike.
template <class T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<_Float16> = 7.0f;

constexpr int kWindow = 512;       // page entries that a workgroup looks up at a time
constexpr int kTileKeys = 32;
constexpr int kMinChunk = 256;     // keys of a split at least (a split's fixed cost: launch slot, partial result, its share of the join)

__device__ __forceinline__ int split_chunk(int n, int splits) {
  const int c = (n + splits - 1) / splits;
  return max((c + 127) & ~127, kMinChunk);
}

struct Unit {
  int b, t, h, rb, n;  // n: virtual keys
  const int* sel;
};
__device__ __forceinline__ Unit unit_of(const AttArgs& a, int unit) {
  Unit u;
  u.rb = unit % a.row_blocks;
  int x = unit / a.row_blocks;
  u.h = x % a.H;
  x /= a.H;
  if (a.selected) {
    u.t = x % a.T;
    u.b = x / a.T;
    u.sel = a.selected + (((long long)u.b * a.T + u.t) * a.H + u.h) * a.count;
    u.n = a.lengths[u.b] > 0 ? a.count << a.pshift : 0;
  } else {
    u.t = 0;
    u.b = x;
    u.sel = nullptr;
    u.n = max(0, min(a.lengths[u.b], a.slots << a.pshift));
  }
  return u;
}
// query / output row r of a unit, as an offset of its first channel
__device__ __forceinline__ long long row_offset(const AttArgs& a, const Unit& u, int r) {
  const int t = a.selected ? u.t : r / a.G, g = a.selected ? r : r % a.G;
  return (((long long)u.b * a.T + t) * a.heads + (long long)u.h * a.G + g) * a.hd;
}

template <class T, int W, int RT>
__global__ __launch_bounds__(256) void k_paged_attention(AttArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NC = W / 16;                                     // channel tiles
  constexpr int NQ = F32 ? W / 16 : (W >= 32 ? W / 32 : 1);      // key-row operands per 16 keys
  constexpr int ROWS = 16 * RT;
  __shared__ int s_page[kWindow], s_valid[kWindow];
  __shared__ float s_m[4][ROWS], s_l[4][ROWS];
  __shared__ float s_o[2][ROWS][W + 4];

  const int split = blockIdx.x % a.splits;
  const Unit u = unit_of(a, blockIdx.x / a.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
  const int chunk = split_chunk(u.n, a.splits);
  const int begin = split * chunk, end = min(u.n, begin + chunk);
  if (begin >= end && split > 0) return;  // (the join knows how many splits a unit has)
  const int P = 1 << a.pshift;
  const long long head_stride = (long long)P * W, page_stride = head_stride * a.H;
  const T* __restrict__ keys = (const T*)a.keys + u.h * head_stride;
  const T* __restrict__ values = (const T*)a.values + u.h * head_stride;

  // query operands: row r16 of each row tile, channels as the key rows' loads deal them out
  uint4 qf[RT][NQ];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = (u.rb * RT + rt) * 16 + r16;
    const T* qr = (const T*)a.q + (r < a.rows ? row_offset(a, u, r) : 0);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      constexpr int PER = F32 ? 4 : (W >= 32 ? 8 : 4);
      union {
        T v[16 / sizeof(T)];
        uint4 u4;
      } x;
      x.u4 = uint4{0, 0, 0, 0};
      const int c0 = F32 ? 16 * i + 4 * g : (W >= 32 ? 32 * i + 8 * g : 4 * g);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (r < a.rows && c0 + j < a.hd) x.v[j] = qr[c0 + j];
      qf[rt][i] = x.u4;
    }
  }

  f32x4 o[RT][NC];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -FLT_MAX;
    l[rt] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[rt][c] = f32x4{0, 0, 0, 0};
  }

  const int e_begin = begin >> a.pshift, e_end = (end + P - 1) >> a.pshift;
  for (int e0 = e_begin; e0 < e_end; e0 += kWindow) {
    const int ne = min(kWindow, e_end - e0);
    if (e0 != e_begin) __syncthreads();
    for (int i = threadIdx.x; i < ne; i += 256) {
      const int logical = u.sel ? u.sel[e0 + i] : e0 + i;
      int page = -1, valid = 0;
      if (logical >= 0 && logical < a.slots) page = a.table[(long long)u.b * a.slots + logical];
      if (page >= 0 && page < a.num_pages) valid = min(max(a.lengths[u.b] - (logical << a.pshift), 0), P);
      else page = 0;
      s_page[i] = page;
      s_valid[i] = valid;
    }
    __syncthreads();
    const int w_begin = max(begin, e0 << a.pshift), w_end = min(end, (e0 + ne) << a.pshift);
    for (int base = w_begin + wave * kTileKeys; base < w_end; base += 4 * kTileKeys) {
      // this lane's key row and value group; a group of 8 (4) keys lies in one page
      f32x4 s[RT][2];
      int left[2];  // valid keys of the lane's score group(s)
      if constexpr (F32) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int i = base + 16 * t, e = min((i >> a.pshift) - e0, ne - 1), off = i & (P - 1);
          left[t] = i < w_end ? s_valid[e] - off - 4 * g : 0;
          const T* kr = keys + s_page[e] * page_stride + (long long)(off + r16) * W + 4 * g;
          f32x4 kf[NQ];
#pragma unroll
          for (int j = 0; j < NQ; ++j) kf[j] = *reinterpret_cast<const f32x4*>(kr + 16 * j);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              const f32x4 qv = __builtin_bit_cast(f32x4, qf[rt][j]);
#pragma unroll
              for (int x = 0; x < 4; ++x) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][x], qv[x], acc, 0, 0, 0);
            }
            s[rt][t] = acc;
          }
        }
      } else {
        const int ik = base + 8 * (r16 >> 2), ek = min((ik >> a.pshift) - e0, ne - 1), offk = (ik & (P - 1)) + (r16 & 3);
        const T* kr = keys + s_page[ek] * page_stride + (long long)offk * W;
        const int iv = base + 8 * g, ev = min((iv >> a.pshift) - e0, ne - 1);
        left[0] = iv < w_end ? s_valid[ev] - (iv & (P - 1)) : 0;
        left[1] = left[0] - 4;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if constexpr (W >= 32) {
            uint4 kf[NQ];
#pragma unroll
            for (int j = 0; j < NQ; ++j) kf[j] = *reinterpret_cast<const uint4*>(kr + 4 * t * W + 32 * j + 8 * g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              f32x4 acc = {0, 0, 0, 0};
#pragma unroll
              for (int j = 0; j < NQ; ++j)
                acc = Mma<T>::k32(__builtin_bit_cast(typename Mma<T>::V8, kf[j]), __builtin_bit_cast(typename Mma<T>::V8, qf[rt][j]), acc);
              s[rt][t] = acc;
            }
          } else {
            const uint2 kf = *reinterpret_cast<const uint2*>(kr + 4 * t * W + 4 * g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][t] = Mma<T>::k16(kf, uint2{qf[rt][0].x, qf[rt][0].y}, f32x4{0, 0, 0, 0});
          }
        }
      }
      const bool ragged = __any(left[0] < 4 || left[1] < 4);
      if (ragged && !__any(left[0] > 0 || left[1] > 0)) continue;  // nothing of this tile is there

      // scores in base-2 logarithms; keys that are not there at -inf, whatever their slots hold
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float v = s[rt][t][x] * a.scale_log2;
            if (ragged) v = x < left[t] ? v : -INFINITY;
            s[rt][t][x] = v;
            top = fmaxf(top, v);
          }
        // the maximum is moved only when a score passes it by 8 (a weight of 256, harmless in 32 bits): rarely after the first tile
        if (__any(top > m[rt] + 8.0f)) {
          float nm = fmaxf(top, __shfl_xor(top, 16));
          nm = fmaxf(nm, __shfl_xor(nm, 32));
          nm = fmaxf(nm, m[rt]);
          const float f = __builtin_amdgcn_exp2f(m[rt] - nm);
          m[rt] = nm;
          l[rt] *= f;
#pragma unroll
          for (int c = 0; c < NC; ++c) o[rt][c] *= f;
        }
        const float base_m = m[rt] - kLift<T>;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s[rt][t][x] = __builtin_amdgcn_exp2f(s[rt][t][x] - base_m);
            l[rt] += s[rt][t][x];
          }
      }

      if constexpr (F32) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int i = base + 16 * t, e = min((i >> a.pshift) - e0, ne - 1), off = (i & (P - 1)) + 4 * g;
          const T* vr = values + s_page[e] * page_stride + (long long)r16 * P + off;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            f32x4 vf = *reinterpret_cast<const f32x4*>(vr + (long long)16 * c * P);
            if (ragged) {
#pragma unroll
              for (int x = 0; x < 4; ++x) vf[x] = x < left[t] ? vf[x] : 0.0f;  // a weight of zero does not hide a NaN
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[rt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[x], s[rt][t][x], o[rt][c], 0, 0, 0);
          }
        }
      } else {
        // the weights go to the matrix cores as two 16-bit values each (high part and rest): the sum keeps 16 bits and more of every
        // weight, so that the output's own rounding is the only one of its size
        typename Mma<T>::V8 ph[RT], pl[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float p = s[rt][x >> 2][x & 3];
            const T hi = stored<T>(p);
            ph[rt][x] = hi;
            pl[rt][x] = (T)(p - (float)hi);
          }
        const int iv = base + 8 * g, ev = min((iv >> a.pshift) - e0, ne - 1);
        const T* vr = values + s_page[ev] * page_stride + (long long)r16 * P + (iv & (P - 1));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          typename Mma<T>::V8 vf = __builtin_bit_cast(typename Mma<T>::V8, *reinterpret_cast<const uint4*>(vr + (long long)16 * c * P));
          if (ragged) {
#pragma unroll
            for (int x = 0; x < 8; ++x) vf[x] = x < left[0] ? vf[x] : (T)0.0f;
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            o[rt][c] = Mma<T>::k32(vf, ph[rt], o[rt][c]);
            o[rt][c] = Mma<T>::k32(vf, pl[rt], o[rt][c]);
          }
        }
      }
    }
  }

  // the four waves' results onto a common maximum, then added in a fixed order: (0 + 2) + (1 + 3)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    if (g == 0) s_m[wave][rt * 16 + r16] = m[rt];
  }
  __syncthreads();
  float gm[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + r16;
    gm[rt] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float f = __builtin_amdgcn_exp2f(m[rt] - gm[rt]);
    l[rt] *= f;
    if (g == 0) s_l[wave][r] = l[rt];
#pragma unroll
    for (int c = 0; c < NC; ++c) o[rt][c] *= f;
  }
  auto put = [&](int slab) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(&s_o[slab][rt * 16 + r16][16 * c + 4 * g]) = o[rt][c];
  };
  auto add = [&](int slab) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int c = 0; c < NC; ++c) o[rt][c] += *reinterpret_cast<const f32x4*>(&s_o[slab][rt * 16 + r16][16 * c + 4 * g]);
  };
  if (wave >= 2) put(wave - 2);
  __syncthreads();
  if (wave < 2) add(wave);
  __syncthreads();
  if (wave == 1) put(0);
  __syncthreads();
  if (wave != 0) return;
  add(0);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + r16;
    l[rt] = (s_l[0][r] + s_l[2][r]) + (s_l[1][r] + s_l[3][r]);
  }
  const bool alone = u.n <= chunk;  // this split is the unit's only one: no join
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = (u.rb * RT + rt) * 16 + r16;
    if (alone) {
      if (r < a.rows) {
        // no token at all (an empty context, or no selected page holds one): zeros, not 0 / 0
        const float inv = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
        T* out = (T*)a.out + row_offset(a, u, r);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (16 * c + 4 * g + x < a.hd) out[16 * c + 4 * g + x] = (T)(o[rt][c][x] * inv);
      }
    } else {
      const long long slot = (long long)blockIdx.x * ROWS + rt * 16 + r16;
#pragma unroll
      for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(a.part + slot * W + 16 * c + 4 * g) = o[rt][c];
      if (g == 0) {
        float* ml = a.part + (long long)gridDim.x * ROWS * W + slot * 2;
        ml[0] = gm[rt];
        ml[1] = l[rt];
      }
    }
  }
}

// The join of a row's splits: one workgroup a row, 256 / (W / 4) splits at a time, sums in a fixed order.
template <class T, int W>
__global__ __launch_bounds__(256) void k_paged_join(AttArgs a, int rows_per_block, int blocks) {
  constexpr int L = W / 4, N = 256 / L;
  __shared__ f32x4 s_o[N][L];
  __shared__ float s_l[N];
  const int r_in = blockIdx.x % a.rows, rest = blockIdx.x / a.rows;  // rest = unit without its row block
  const int unit = rest * a.row_blocks + r_in / rows_per_block;
  const Unit u = unit_of(a, unit);
  const int chunk = split_chunk(u.n, a.splits);
  if (u.n <= chunk) return;
  const int ns = (u.n + chunk - 1) / chunk;
  const float* ml = a.part + (long long)blocks * rows_per_block * W;
  const long long first = ((long long)unit * a.splits) * rows_per_block + r_in % rows_per_block;
  float top = -FLT_MAX;
  for (int s = threadIdx.x & 63; s < ns; s += 64) top = fmaxf(top, ml[(first + (long long)s * rows_per_block) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const int c = threadIdx.x % L, n = threadIdx.x / L;
  f32x4 acc = {0, 0, 0, 0};
  float l = 0.0f;
  if (n < N)
    for (int s = n; s < ns; s += N) {
      const long long slot = first + (long long)s * rows_per_block;
      const float f = __builtin_amdgcn_exp2f(ml[slot * 2] - top);
      l += f * ml[slot * 2 + 1];
      acc += f * *reinterpret_cast<const f32x4*>(a.part + slot * W + 4 * c);
    }
  if (n < N) {
    s_o[n][c] = acc;
    if (c == 0) s_l[n] = l;
  }
  __syncthreads();
  if (threadIdx.x < L) {
    float sum = 0.0f;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
      sum += s_l[i];
      v += s_o[i][c];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = (T*)a.out + row_offset(a, u, r_in);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (4 * c + x < a.hd) out[4 * c + x] = (T)(v[x] * inv);
  }
}

// ---- selection of pages -----------------------------------------------------------------------------------------------------------------
// score of a page for a query row: sum_c max(q_c, 0) key_max_c + min(q_c, 0) key_min_c >= q . k for every key of the page; a key-value
// head's score is the largest of the G rows that share it.  In 64 bits: the choice is a border between nearly equal numbers, and must not
// depend on the order of a sum.
struct SelectArgs {
  const void *q, *kmin, *kmax;
  const int *table, *lengths;
  int B, T, heads, H, G, hd, W, slots, num_pages, pshift, count;
  int score_blocks, score_steps;  // workgroups of a (context, head), steps of each
  double* scores;  // [B, T, H, slots]; -inf: the page is not there (entries behind the context's last page are not written)
  int* out;        // [B, T, H, count]
};

// One summary is read once: W / 8 lanes take 8 channels of a page each, 64 / that many pages side by side in a wave, two steps of them
// at a time, all query rows over them.  The lanes' sums meet in a rotation within the 16-lane row, whose result is the same in
// every lane.  (The 64-bit matrix instruction reaches 42 TFLOP/s here and pays for 16 rows whatever their number; four rows on
// the vector unit cost less than the read.)
template <int N>
__device__ __forceinline__ double row_rotate(double x) {  // the value N lanes on in the row of 16
  const long long u = __double_as_longlong(x);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)u, 0x120 + N, 0xf, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), 0x120 + N, 0xf, 0xf, false);
  return __longlong_as_double(((long long)hi << 32) | (unsigned)lo);
}
// sum over groups of L neighbouring lanes, in every lane of the group
template <int L>
__device__ __forceinline__ double group_sum(double x) {
  if constexpr (L >= 16) {
    x += row_rotate<8>(x);
    x += row_rotate<4>(x);
    x += row_rotate<2>(x);
    x += row_rotate<1>(x);
    if constexpr (L == 32) x += __shfl_xor(x, 16);
  } else {
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) x += __shfl_xor(x, d);
  }
  return x;
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    const Pack<T, N> v = reinterpret_cast<const Pack<T, N>*>(p)[i];
#pragma unroll
    for (int j = 0; j < N; ++j) x[N * i + j] = to_f(v.v[j]);
  }
}

constexpr int kScoreRows = 4;  // query rows in registers at a time

struct ScoreQuery {
  double plus[kScoreRows][8], minus[kScoreRows][8];
};
template <class T>
__device__ __forceinline__ void load_query(const SelectArgs& a, int b, int h, int r0, int rows, int c0, ScoreQuery& q) {
#pragma unroll
  for (int r = 0; r < kScoreRows; ++r) {
    const int row = min(r0 + r, rows - 1);
    const T* p = (const T*)a.q + (((long long)b * a.T + row / a.G) * a.heads + (long long)h * a.G + row % a.G) * a.hd;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double x = c0 + j < a.hd ? (double)to_f(p[c0 + j]) : 0.0;
      q.plus[r][j] = x > 0.0 ? x : (x != x ? x : 0.0);
      q.minus[r][j] = x < 0.0 ? x : 0.0;
    }
  }
}

template <class T, int W>
__global__ __launch_bounds__(256) void k_paged_score(SelectArgs a) {
  constexpr int L = W == 96 ? 16 : W / 8, GP = 64 / L, STEP = 2 * GP;
  const int unit = blockIdx.x / a.score_blocks, block = blockIdx.x % a.score_blocks;
  const int h = unit % a.H, b = unit / a.H;
  const int P = 1 << a.pshift;
  const int np = (int)min((long long)a.slots, ((long long)max(a.lengths[b], 0) + P - 1) >> a.pshift);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = (lane % L) * 8, gp = lane / L;
  const int per_block = 4 * STEP * a.score_steps;
  if (block * per_block >= np) return;
  const int rows = a.T * a.G;
  ScoreQuery q;
  load_query<T>(a, b, h, 0, rows, c0, q);
  for (int step = 0; step < a.score_steps; ++step) {
    const int first = block * per_block + (step * 4 + wave) * STEP;
    if (first >= np) break;
    double mx[2][8], mn[2][8];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int slot = first + i * GP + gp;
      const int page = slot < np ? a.table[(long long)b * a.slots + slot] : -1;
      there[i] = page >= 0 && page < a.num_pages;
      float x[8];
      const long long at = ((long long)(there[i] ? page : 0) * a.H + h) * W + c0;
      if (W != 96 || c0 < W) load8((const T*)a.kmax + at, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) mx[i][j] = W != 96 || c0 < W ? (double)x[j] : 0.0;
      if (W != 96 || c0 < W) load8((const T*)a.kmin + at, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) mn[i][j] = W != 96 || c0 < W ? (double)x[j] : 0.0;
    }
    double best[2] = {-INFINITY, -INFINITY};
    for (int r0 = 0; r0 < rows; r0 += kScoreRows) {
      if (rows > kScoreRows) load_query<T>(a, b, h, r0, rows, c0, q);
#pragma unroll
      for (int r = 0; r < kScoreRows; ++r) {
        if (r0 + r >= rows) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          double s = 0.0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            s = fma(q.plus[r][j], mx[i][j], s);
            s = fma(q.minus[r][j], mn[i][j], s);
          }
          s = group_sum<L>(s);
          best[i] = (s > best[i] || s != s) ? s : best[i];
        }
        const int row = r0 + r;
        if (row % a.G == a.G - 1) {
          const int t = row / a.G;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int slot = first + i * GP + gp;
            if (slot < np && lane % L == 0) a.scores[(((long long)b * a.T + t) * a.H + h) * a.slots + slot] = there[i] ? best[i] : -INFINITY;
            best[i] = -INFINITY;
          }
        }
      }
    }
  }
}

// order-preserving key: larger score, larger key; NaN above all; -inf (not there) at kNotThere, below all others
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return ~0ull;
  unsigned long long u = __double_as_longlong(s + 0.0);  // (-0 and 0 are equal)
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
constexpr unsigned long long kNotThere = 0x000fffffffffffffull;  // score_key(-inf)

// The count best of a row, the lowest slots first among equals, written in ascending order.  A threshold bucket is found by histogram
// over [smallest, largest] key of the candidates: first over the scores themselves (2048 equal steps: scores spread over them whatever
// their scale), then, in the bucket that holds the border, over the keys as integers, each time from their highest differing bit: 11 bits
// a pass, so it ends.  Then one ordered pass writes what lies above the bucket, and of the last bucket's equals the first `need`.
constexpr int kBuckets = 2048;
__global__ __launch_bounds__(1024) void k_paged_select(SelectArgs a) {
  __shared__ int s_hist[kBuckets];
  __shared__ unsigned long long s_lo[16], s_hi[16];
  __shared__ int s_sum[16], s_bin, s_above;
  __shared__ int s_wave[2][16];
  const long long row = blockIdx.x;
  const int b = (int)(row / ((long long)a.T * a.H));
  const double* __restrict__ sc = a.scores + row * a.slots;
  int* __restrict__ out = a.out + row * a.count;
  const int P = 1 << a.pshift;
  const int np = (int)min((long long)a.slots, ((long long)max(a.lengths[b], 0) + P - 1) >> a.pshift);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int R = 4;  // scores that a thread keeps (rows of up to 4096 pages are read once)
  double mine[R];
#pragma unroll
  for (int i = 0; i < R; ++i) mine[i] = tid + 1024 * i < np ? sc[tid + 1024 * i] : -INFINITY;
  auto score = [&](int i) { return i < R ? (i == 0 ? mine[0] : i == 1 ? mine[1] : i == 2 ? mine[2] : mine[3]) : sc[tid + 1024 * i]; };
  const int mine_n = np > tid ? (np - tid + 1023) / 1024 : 0;

  // candidates: keys in [lo, hi]; everything above hi is taken
  unsigned long long lo = kNotThere + 1, hi = ~0ull;
  int need = a.count;
  bool all = false, exact = false;
  for (int pass = 0;; ++pass) {
    unsigned long long mn = ~0ull, mx = 0;
    int n = 0;
    for (int i = 0; i < mine_n; ++i) {
      const unsigned long long k = score_key(score(i));
      if (k >= lo && k <= hi) {
        mn = min(mn, k);
        mx = max(mx, k);
        ++n;
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      mn = min(mn, (unsigned long long)__shfl_xor((long long)mn, d));
      mx = max(mx, (unsigned long long)__shfl_xor((long long)mx, d));
      n += __shfl_xor(n, d);
    }
    if (lane == 0) {
      s_lo[wave] = mn;
      s_hi[wave] = mx;
      s_sum[wave] = n;
    }
    for (int i = tid; i < kBuckets; i += 1024) s_hist[i] = 0;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      mn = min(mn, s_lo[w]);
      mx = max(mx, s_hi[w]);
      n += s_sum[w];
    }
    if (n <= need) {  // all candidates
      all = true;
      if (n > 0) lo = mn;
      break;
    }
    lo = mn;
    hi = mx;
    if (mn == mx) {  // equals: the first `need` of them
      exact = true;
      break;
    }
    const unsigned long long kInfKey = 0xfff0000000000000ull, kLowKey = kNotThere + 1;
    const bool linear = pass == 0 && mx < kInfKey && mn >= kLowKey;  // (finite scores)
    const double base = linear ? __longlong_as_double((mn >> 63) ? (long long)(mn & 0x7fffffffffffffffull) : (long long)~mn) : 0.0;
    const double top = linear ? __longlong_as_double((mx >> 63) ? (long long)(mx & 0x7fffffffffffffffull) : (long long)~mx) : 0.0;
    const double inv = linear ? (double)(kBuckets - 1) / (top - base) : 0.0;
    const int shift = max(0, 64 - __clzll((long long)(mx - mn)) - 11);
    // (a step that is no number, or infinite: all in one bucket, and the next pass goes by the integers)
    auto bucket = [&](double s, unsigned long long k) { return linear ? min(max((int)((s - base) * inv), 0), kBuckets - 1) : (int)((k - mn) >> shift); };
    for (int i = 0; i < mine_n; ++i) {
      const double s = score(i);
      const unsigned long long k = score_key(s);
      if (k >= lo && k <= hi) atomicAdd(&s_hist[bucket(s, k)], 1);
    }
    __syncthreads();
    // the bucket that holds the border: counts from the top, two buckets a thread
    const int b1 = kBuckets - 1 - 2 * tid, h1 = s_hist[b1], h0 = s_hist[b1 - 1];
    int upto = h1 + h0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += s_sum[w];
    const int before = upto - h1 - h0;
    if (before < need && upto >= need) {
      s_bin = before + h1 >= need ? b1 : b1 - 1;
      s_above = before + h1 >= need ? before : before + h1;
    }
    __syncthreads();
    const int bin = s_bin;
    need -= s_above;
    // the bucket's own smallest and largest key are the next candidates' (found by the next pass's reduction)
    unsigned long long bl = ~0ull, bh = 0;
    for (int i = 0; i < mine_n; ++i) {
      const double s = score(i);
      const unsigned long long k = score_key(s);
      if (k >= lo && k <= hi && bucket(s, k) == bin) {
        bl = min(bl, k);
        bh = max(bh, k);
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      bl = min(bl, (unsigned long long)__shfl_xor((long long)bl, d));
      bh = max(bh, (unsigned long long)__shfl_xor((long long)bh, d));
    }
    __syncthreads();
    if (lane == 0) {
      s_lo[wave] = bl;
      s_hi[wave] = bh;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      bl = min(bl, s_lo[w]);
      bh = max(bh, s_hi[w]);
    }
    lo = bl;
    hi = bh;
    __syncthreads();
  }
  // above hi: taken; in [lo, hi]: all of them, or the first `need`
  int base_m = 0, base_t = 0;
  for (int i = 0; i * 1024 < np; ++i) {
    const int slot = i * 1024 + tid;
    bool sure = false, maybe = false;
    if (slot < np) {
      const unsigned long long k = score_key(score(i));
      if (k > kNotThere) {
        sure = k > hi || (all && k >= lo);
        maybe = exact && k == lo;
      }
    }
    const unsigned long long below = (1ull << lane) - 1, bm = __ballot(maybe), bs = __ballot(sure);
    if (lane == 0) {
      s_wave[0][wave] = __popcll(bm);
      s_wave[1][wave] = __popcll(bs);
    }
    __syncthreads();
    int m = base_m, t = base_t, bm_all = 0, bs_all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w < wave) {
        m += s_wave[0][w];
        t += s_wave[1][w];
      }
      bm_all += s_wave[0][w];
      bs_all += s_wave[1][w];
    }
    m += __popcll(bm & below);
    t += __popcll(bs & below);
    // (of the equals before this slot, those that were taken: the first `need`)
    const int at = t + min(m, exact ? need : 0);
    if ((sure || (maybe && m < need)) && at < a.count) out[at] = slot;
    base_m += bm_all;
    base_t += bs_all;
    __syncthreads();
  }
  for (int i = base_t + min(base_m, exact ? need : 0) + tid; i < a.count; i += 1024) out[i] = -1;
}

template <class TI, class T, int VEC, int VT>
void append_go(const AppendArgs& a, int units, hipStream_t s) {
  k_paged_append<TI, T, VEC, VT><<<dim3(units, (a.H + a.heads_per_wg - 1) / a.heads_per_wg), 256, 0, s>>>(a);
}

template <class TI, class T>
void append_typed(AppendArgs& a, int units, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T), VT = VEC;  // 16-byte stores both ways
  // wide loads need every chunk at a multiple of its size
  const uintptr_t align = sizeof(TI) * VEC < 16 ? sizeof(TI) * VEC : 16;
  const bool wide = a.hd % VEC == 0 && a.k_stride % VEC == 0 && a.v_stride % VEC == 0 && (uintptr_t)a.k % align == 0 && (uintptr_t)a.v % align == 0;
  if (wide)
    append_go<TI, T, VEC, VT>(a, units, s);
  else
    append_go<TI, T, 1, VT>(a, units, s);
}

template <class T, int W, int RT>
void attention_go(const AttArgs& a, int blocks, hipStream_t s) {
  k_paged_attention<T, W, RT><<<blocks, 256, 0, s>>>(a);
  if (a.splits > 1) {
    const int rows = blocks / a.splits / a.row_blocks * a.rows;
    k_paged_join<T, W><<<rows, 256, 0, s>>>(a, 16 * RT, blocks);
  }
}
template <class T>
int attention_typed(const AttArgs& a, int W, int RT, int blocks, hipStream_t s) {
  switch (W) {
    case 16: RT == 2 ? attention_go<T, 16, 2>(a, blocks, s) : attention_go<T, 16, 1>(a, blocks, s); return 0;
    case 32: RT == 2 ? attention_go<T, 32, 2>(a, blocks, s) : attention_go<T, 32, 1>(a, blocks, s); return 0;
    case 64: RT == 2 ? attention_go<T, 64, 2>(a, blocks, s) : attention_go<T, 64, 1>(a, blocks, s); return 0;
    case 96: RT == 2 ? attention_go<T, 96, 2>(a, blocks, s) : attention_go<T, 96, 1>(a, blocks, s); return 0;
    case 128: RT == 2 ? attention_go<T, 128, 2>(a, blocks, s) : attention_go<T, 128, 1>(a, blocks, s); return 0;
    case 256: attention_go<T, 256, 1>(a, blocks, s); return 0;
  }
  return 1;
}

template <class T>
void score_typed(const SelectArgs& a, int blocks, hipStream_t s) {
  switch (a.W) {
    case 16: k_paged_score<T, 16><<<blocks, 256, 0, s>>>(a); break;
    case 32: k_paged_score<T, 32><<<blocks, 256, 0, s>>>(a); break;
    case 64: k_paged_score<T, 64><<<blocks, 256, 0, s>>>(a); break;
    case 96: k_paged_score<T, 96><<<blocks, 256, 0, s>>>(a); break;
    case 128: k_paged_score<T, 128><<<blocks, 256, 0, s>>>(a); break;
    default: k_paged_score<T, 256><<<blocks, 256, 0, s>>>(a); break;
  }
}

// rows of a unit go 16 or 32 at a time (one or two row tiles share a pass over the keys); heads of 256 channels leave registers for 16
int row_tiles(int rows, int W) { return rows > 16 && W < 256 ? 2 : 1; }

struct AttPlan {
  long long units;
  int row_blocks, splits, RT;
};
// Workgroups for 256 CUs: a unit's keys are split until there are about kTargetWgs of them, kMinChunk keys each at least.
constexpr int kTargetWgs = 2048;
AttPlan attention_plan(int B, int T, int H, int G, int W, long long capacity, bool selected) {
  AttPlan p;
  const int rows = selected ? G : T * G;
  p.RT = row_tiles(rows, W);
  p.row_blocks = (rows + 16 * p.RT - 1) / (16 * p.RT);
  p.units = (long long)B * (selected ? T : 1) * H * p.row_blocks;
  const long long most = std::max(1LL, (capacity + kMinChunk - 1) / kMinChunk);
  p.splits = (int)std::min(most, std::max(1LL, kTargetWgs / std::max(1LL, p.units)));
  return p;
}

}  // namespace

int paged_width(int head_dim) {
  for (int w : {16, 32, 64, 96, 128, 256})
    if (head_dim >= 1 && head_dim <= w) return w;
  return 0;
}

int launch_paged_append(const void* k, long long k_stride, const void* v, long long v_stride, int in_type, int n_tokens, const float* positions,
                        int axes, int rotary, double base, const int* offsets, const int* starts, const int* table, int B, int slots, int pshift,
                        int H, int hd, int num_pages, int type, void* keys, void* values, void* kmin, void* kmax, hipStream_t s) {
  AppendArgs a{};
  a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride;
  a.positions = positions, a.axes = axes, a.rotary = rotary, a.log2_base = std::log2(base);
  a.offsets = offsets, a.starts = starts, a.table = table, a.B = B, a.slots = slots, a.n_tokens = n_tokens, a.pshift = pshift;
  a.H = H, a.hd = hd, a.W = paged_width(hd), a.num_pages = num_pages;
  a.keys = keys, a.values = values, a.kmin = kmin, a.kmax = kmax;
  // (context, page) pairs: each holds a token, and a context has at most two pages more than its tokens fill
  const int units = (int)std::min<long long>(n_tokens, (n_tokens >> pshift) + 2LL * B);
  const int parts = std::min(H, std::max(1, 1024 / units));
  a.heads_per_wg = (H + parts - 1) / parts;
  if (type == 0 && in_type == 0) append_typed<float, float>(a, units, s);
  else if (type == 1 && in_type == 0) append_typed<float, _Float16>(a, units, s);
  else if (type == 2 && in_type == 0) append_typed<float, __bf16>(a, units, s);
  else if (type == 1 && in_type == 1) append_typed<_Float16, _Float16>(a, units, s);
  else if (type == 2 && in_type == 2) append_typed<__bf16, __bf16>(a, units, s);
  else return 1;
  return 0;
}

long long paged_attention_workspace_floats(int B, int T, int H, int G, int hd, long long capacity, bool selected) {
  const int W = paged_width(hd);
  const AttPlan p = attention_plan(B, T, H, G, W, capacity, selected);
  return p.splits > 1 ? p.units * p.splits * 16 * p.RT * (W + 2) : 0;
}

int launch_paged_attention(const void* q, const void* keys, const void* values, int type, const int* table, const int* lengths, const int* selected,
                           int count, int B, int T, int H, int G, int hd, int slots, int num_pages, int pshift, float scale, void* out, float* work,
                           hipStream_t s) {
  const int W = paged_width(hd);
  const AttPlan p = attention_plan(B, T, H, G, W, (long long)(selected ? count : slots) << pshift, selected != nullptr);
  if (p.units * p.splits > 0x7fffffffLL || p.units / p.row_blocks * (selected ? G : T * G) > 0x7fffffffLL) return 2;
  AttArgs a{};
  a.q = q, a.keys = keys, a.values = values, a.table = table, a.lengths = lengths, a.selected = selected;
  a.B = B, a.T = T, a.heads = H * G, a.H = H, a.G = G, a.hd = hd, a.slots = slots, a.num_pages = num_pages, a.pshift = pshift, a.count = count;
  a.rows = selected ? G : T * G, a.row_blocks = p.row_blocks, a.splits = p.splits;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.out = out, a.part = work;
  const int blocks = (int)(p.units * p.splits);
  if (type == 0) return attention_typed<float>(a, W, p.RT, blocks, s);
  if (type == 1) return attention_typed<_Float16>(a, W, p.RT, blocks, s);
  return attention_typed<__bf16>(a, W, p.RT, blocks, s);
}

long long paged_select_workspace_doubles(int B, int T, int H, int slots) { return (long long)B * T * H * slots; }

int launch_paged_select(const void* q, const void* kmin, const void* kmax, int type, const int* table, const int* lengths, int B, int T, int H, int G,
                        int hd, int slots, int num_pages, int pshift, int count, double* work, int* out, hipStream_t s) {
  if ((long long)B * T * H > 0x7fffffffLL || (long long)T * G > 0x7fffffffLL) return 2;
  SelectArgs a{};
  a.q = q, a.kmin = kmin, a.kmax = kmax, a.table = table, a.lengths = lengths;
  a.B = B, a.T = T, a.heads = H * G, a.H = H, a.G = G, a.hd = hd, a.W = paged_width(hd), a.slots = slots, a.num_pages = num_pages, a.pshift = pshift;
  a.count = count, a.scores = work, a.out = out;
  const int L = a.W == 96 ? 16 : a.W / 8, per_step = 4 * 2 * (64 / L);  // pages of a workgroup's step
  const long long all_steps = (long long)B * H * ((slots + per_step - 1) / per_step);
  a.score_steps = (int)std::min(16LL, std::max(1LL, all_steps / 2048));  // about 8 workgroups a CU, each with its query loaded once
  a.score_blocks = (slots + per_step * a.score_steps - 1) / (per_step * a.score_steps);
  if ((long long)B * H * a.score_blocks > 0x7fffffffLL) return 2;
  const int blocks = B * H * a.score_blocks;
  if (type == 0) score_typed<float>(a, blocks, s);
  else if (type == 1) score_typed<_Float16>(a, blocks, s);
  else score_typed<__bf16>(a, blocks, s);
  k_paged_select<<<B * T * H, 1024, 0, s>>>(a);
  return 0;
}

}  // namespace mmf
