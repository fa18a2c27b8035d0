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
#include <numeric>

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
__device__ __forceinline__ float smaller(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// ---- append ---------------------------------------------------------------------------------------------------------------------------
// Token i of the rows offsets[b] .. offsets[b + 1] - 1 becomes token starts[b] + i - offsets[b] of context b.  A workgroup owns one
// (context, page) pair and a range of heads, so a page's summary has one writer and needs no atomics; it finds its pair by a scan over
// the contexts' page counts.  A thread takes VEC channels of VT neighbouring slots: the keys go out row by row as they came, the values
// are transposed in its registers so that both stores are wide.  Large appends of whole 16-byte heads are bound by memory: 138 us for 145 000
// tokens of 8 heads of 64 (float16, 599 MB: 4.3 TB/s).  Heads of 15 are not: 40 us for 55 000 tokens of 8 of them (float32, 107 MB, all of it moved
// once), where 120 of 256 threads have a chunk and a page's rows are asked for behind offsets, table entry, positions and angles.  Single tokens are
// bound by that chain (6 us), those of many contexts by it and by their values: 2 bytes each, every one in a 32-byte piece of its own (12 us for 256
// contexts of 8 heads of 128: 262 144 such pieces).
struct AppendArgs {
  const void *k, *v;
  long long k_stride, v_stride;  // below 2^23
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

// The unit-th (context, page) pair that gets tokens: contexts in order, pages in order.  One thread a context, a scan over the
// workgroup.
__device__ __forceinline__ bool find_segment(const AppendArgs& a, int unit, Segment& s) {
  __shared__ int s_total[4], s_seg[5];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << a.pshift;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 256) {
    const int b = b0 + tid;
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
    if (lane == 63) s_total[wave] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) upto += s_total[w];
      all += s_total[w];
    }
    if (before + all > unit) {
      if (before + upto > unit && before + upto - np <= unit) {
        const int slot = (st >> a.pshift) + unit - (before + upto - np), page_first = slot << a.pshift, first = max(st - page_first, 0);
        s_seg[0] = b;
        s_seg[1] = slot;
        s_seg[2] = first;
        s_seg[3] = min(st + n - page_first, P);
        s_seg[4] = lo + page_first + first - st;
      }
      __syncthreads();
      s.b = s_seg[0], s.slot = s_seg[1], s.first = s_seg[2], s.last = s_seg[3], s.row = s_seg[4];
      return true;
    }
    before += all;
    __syncthreads();
  }
  return false;
}

// A thread takes VEC channels of VT slots.  KIND 2: the heads are whole chunks, everything moves in 16-byte pieces; 1: chunks of the row
// that may belong to two heads, whose rotation pairs are still the lane's own (the policy's heads of 15); 0: any layout, one channel,
// its partner read beside it.  The page is taken in blocks of tokens whose cos / sin fit into LDS: computed once for all heads (of the row's
// own pairs where the code covers the whole row), at [slot of a group][chunk of pairs][group], the order in which lanes read them.
// KIND 1 puts the block's keys together in LDS and stores them from there in 16-byte pieces of the pages, padding included (stored
// as the lanes have them, 4 + 12 bytes or 4 times 4, the keys took 11 us of 43 for 32 contexts of 8 heads of 15).
template <int KIND>
constexpr int kAppendRow = KIND == 1 ? 256 : 1024;  // channels of a workgroup at most
template <class TI, class T, int KIND>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  constexpr int VT = 16 / sizeof(T), VEC = KIND ? VT : 1, NP = VEC > 1 ? VEC / 2 : 1;
  constexpr int kAngles = sizeof(T) == 4 ? 2048 : 4096;  // (the 32-bit kernels have the registers for more workgroups a CU than 32 KB leave room for)
  __shared__ __attribute__((aligned(16))) float2 s_angle[kAngles];
  constexpr int ROW = kAppendRow<KIND>, kTile = KIND == 1 ? 4096 * 4 / sizeof(T) : 0;
  __shared__ double s_turns[ROW / 2 + 8];           // turns a unit of position, by pair
  __shared__ float s_lo[ROW], s_hi[ROW];
  __shared__ __attribute__((aligned(16))) T s_tile[KIND == 1 ? kTile : 1];  // [slot of the block][channel of the workgroup]
  Segment seg;
  if (!find_segment(a, blockIdx.x, seg)) return;
  const int page = a.table[(long long)seg.b * a.slots + seg.slot];
  if (page < 0 || page >= a.num_pages) return;
  const int tid = threadIdx.x;
  const int h0 = blockIdx.y * a.heads_per_wg, nh = min(a.heads_per_wg, a.H - h0);
  const int c0 = h0 * a.hd, nchunks = nh * a.hd / VEC;
  const bool whole_row = a.rotary > a.hd;
  const int pairs = a.rotary ? (whole_row ? (nh * a.hd + 1 + (c0 & 1)) / 2 : a.rotary / 2) : 0;  // (a whole row's pairs may begin before h0's first channel)
  const int pair0 = whole_row ? c0 / 2 : 0;
  const int span = a.rotary ? a.rotary / a.axes : 2;
  // (bases that are the workgroup's, 32-bit offsets from them: the host checks that a page and 256 rows stay below 2^31 elements)
  const TI* __restrict__ kin = (const TI*)a.k + (long long)seg.row * a.k_stride;
  const TI* __restrict__ vin = (const TI*)a.v + (long long)seg.row * a.v_stride;
  const long long page_head = (long long)page * a.H;
  T* __restrict__ kpage = (T*)a.keys + (page_head << a.pshift) * a.W;
  T* __restrict__ vpage = (T*)a.values + (page_head << a.pshift) * a.W;
  for (int i = tid; i < pairs; i += 256) {
    const int j = (2 * (pair0 + i)) % span;  // pair j / 2 of its axis: position * base^(-j / span) / 2 pi turns
    s_turns[i] = exp2(-a.log2_base * (double)j / (double)span) * 0.15915494309189533576888;
  }
  const int pair_chunks = (pairs + NP - 1) / NP;
  int groups = pairs ? min(256 / VT, kAngles / (pair_chunks * NP * VT)) : 256 / VT;  // of a block
  if (KIND == 1) groups = min(groups, kTile / (nh * a.hd * VT));
  const int block = groups * VT;
  // what the page's summary held (it begins anew with its first slot), asked for early: the first access to a page of a large pool waits long
  constexpr int OLD = ROW / 256;
  const bool merge = seg.first > 0;
  float old_lo[OLD], old_hi[OLD];
  if (merge) {
#pragma unroll
    for (int j = 0; j < OLD; ++j) {
      const int i = min(tid + 256 * j, nh * a.hd - 1);
      const long long at = (page_head + h0 + i / a.hd) * a.W + i % a.hd;
      old_lo[j] = to_f(((const T*)a.kmin)[at]);
      old_hi[j] = to_f(((const T*)a.kmax)[at]);
    }
  }
  bool begun = false;
  for (int first = seg.first / VT * VT; first < seg.last; first += block) {
    const int lo_slot = max(first, seg.first), hi_slot = min(first + block, seg.last);
    if (pairs) {
      __syncthreads();
      const int n = (hi_slot - lo_slot) * pairs;
      for (int i = tid; i < n; i += 256) {
        const int t = i / pairs, w = i - t * pairs, axis = 2 * (pair0 + w) / span, at = lo_slot + t - first;
        const long long row = seg.row + (lo_slot + t - seg.first);
        // taken in turns and reduced in 64 bits (a far position times a frequency loses its fraction in 32), then in 32 on [-1/2, 1/2]
        const double turns = (double)a.positions[row * a.axes + axis] * s_turns[w];
        float2 cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &cs.y, &cs.x);
        s_angle[((at % VT * pair_chunks + w / NP) * groups + at / VT) * NP + w % NP] = cs;
      }
      __syncthreads();
    }
    const int ng = (hi_slot - first + VT - 1) / VT;
    int gw = 1;  // neighbouring lanes take neighbouring slot groups: 8 of them fill the value rows' cache lines
    while (gw < 8 && gw < ng) gw <<= 1;
    const int gl = tid & (gw - 1);
    for (int ch = tid / gw; ch < nchunks; ch += 256 / gw) {
      const int c = c0 + ch * VEC;  // channel in the row
      const int h = c / a.hd, d = c - h * a.hd;
      unsigned kat[1], vat[VEC];  // where slot 0 of channel c (c + i) is in the page's keys (values)
      int pair[NP];                 // its pair in the table, or -1
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int over = KIND == 1 && d + i >= a.hd ? (d + i) / a.hd : 0;
        const int hh = h + over, dd = d + i - over * a.hd;
        if (i == 0) kat[0] = ((unsigned)hh << a.pshift) * a.W + dd;
        vat[i] = ((unsigned)hh * a.W + dd) << a.pshift;
        if (i % 2 == 0) {
          const int w = whole_row ? c + i : dd;
          pair[i / 2] = w < a.rotary ? w / 2 - pair0 : -1;
        }
      }
      float lo[VEC], hi[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        lo[i] = INFINITY;
        hi[i] = -INFINITY;
      }
      for (int g = gl; g < ng; g += gw) {
        const int slot0 = first + g * VT;
        const bool full = slot0 >= seg.first && slot0 + VT <= seg.last;
        // all loads first (a slot outside the block's tokens reads the nearest inside: its values count twice in the summary, which is the same)
        Pack<TI, VEC> kr[VT], vr[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const unsigned row = min(max(slot0 + t, lo_slot), hi_slot - 1) - seg.first;
          kr[t] = *reinterpret_cast<const Pack<TI, VEC>*>(kin + (row * (unsigned)a.k_stride + (unsigned)c));
          vr[t] = *reinterpret_cast<const Pack<TI, VEC>*>(vin + (row * (unsigned)a.v_stride + (unsigned)c));
        }
        Pack<T, VEC> out[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const int slot = min(max(slot0 + t, lo_slot), hi_slot - 1), at = slot - first;
          float x[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) x[i] = to_f(kr[t].v[i]);
          if (pairs) {
            const float2* angle = s_angle + ((at % VT) * pair_chunks * groups + at / VT) * NP;
            if constexpr (VEC > 1) {
              // (branch-free: a pair that is not turned reads some angle and keeps its values)
              Pack<float2, NP> cs;
              if (KIND == 2 || whole_row) {
                cs = *reinterpret_cast<const Pack<float2, NP>*>(angle + max(pair[0], 0) / NP * groups * NP);
              } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) cs.v[i] = angle[max(pair[i], 0) / NP * groups * NP + max(pair[i], 0) % NP];
              }
#pragma unroll
              for (int i = 0; i < NP; ++i) {
                const float e = x[2 * i], o = x[2 * i + 1];
                const float p = e * cs.v[i].x - o * cs.v[i].y, q = o * cs.v[i].x + e * cs.v[i].y;
                x[2 * i] = pair[i] >= 0 ? p : e;
                x[2 * i + 1] = pair[i] >= 0 ? q : o;
              }
            } else if (pair[0] >= 0) {
              const bool odd = (whole_row ? c : d) & 1;
              const float2 cs = angle[pair[0] * groups];
              const float p = to_f(kin[(unsigned)(slot - seg.first) * (unsigned)a.k_stride + (unsigned)c + (odd ? -1 : 1)]);
              x[0] = odd ? x[0] * cs.x + p * cs.y : x[0] * cs.x - p * cs.y;
            }
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            out[t].v[i] = stored<T>(x[i]);  // the one rounding of a key; the summary is of the stored value
            const float y = to_f(out[t].v[i]);
            lo[i] = smaller(lo[i], y);
            hi[i] = larger(hi[i], y);
          }
        }
        if (full) {
#pragma unroll
          for (int t = 0; t < VT; ++t) {
            T* to = kpage + ((unsigned)(slot0 + t) * a.W + kat[0]);
            if (KIND == 1) to = s_tile + (slot0 + t - first) * (nh * a.hd) + ch * VEC;
            *reinterpret_cast<Pack<T, VEC>*>(to) = out[t];
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            Pack<T, VT> col;
#pragma unroll
            for (int t = 0; t < VT; ++t) col.v[t] = (T)to_f(vr[t].v[i]);
            *reinterpret_cast<Pack<T, VT>*>(vpage + (vat[i] + (unsigned)slot0)) = col;
          }
        } else {
#pragma unroll
          for (int t = 0; t < VT; ++t)
            if (slot0 + t >= lo_slot && slot0 + t < hi_slot) {
              T* to = kpage + ((unsigned)(slot0 + t) * a.W + kat[0]);
              if (KIND == 1) to = s_tile + (slot0 + t - first) * (nh * a.hd) + ch * VEC;
              *reinterpret_cast<Pack<T, VEC>*>(to) = out[t];
#pragma unroll
              for (int i = 0; i < VEC; ++i) vpage[vat[i] + (unsigned)(slot0 + t)] = (T)to_f(vr[t].v[i]);
            }
        }
      }
      // over the gw lanes of this chunk, then over the blocks (the first lane of a chunk's group is the same thread in all but a last,
      // shorter block, whose predecessors' results it reads behind a barrier)
      for (int m = 1; m < gw; m <<= 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          lo[i] = smaller(lo[i], __shfl_xor(lo[i], m));
          hi[i] = larger(hi[i], __shfl_xor(hi[i], m));
        }
      }
      if (gl == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s_lo[ch * VEC + i] = begun ? smaller(lo[i], s_lo[ch * VEC + i]) : lo[i];
          s_hi[ch * VEC + i] = begun ? larger(hi[i], s_hi[ch * VEC + i]) : hi[i];
        }
      }
    }
    begun = true;
    __syncthreads();
    if constexpr (KIND == 1) {
      const int wide = (a.hd + VEC - 1) / VEC, each = nh * wide;  // 16-byte pieces of a head, of a slot
      for (int i = tid; i < (hi_slot - lo_slot) * each; i += 256) {
        const int s = i / each, h = (i - s * each) / wide, d = (i - s * each - h * wide) * VEC;
        const T* from = s_tile + (lo_slot + s - first) * (nh * a.hd) + h * a.hd + d;
        Pack<T, VEC> out;
#pragma unroll
        for (int x = 0; x < VEC; ++x) out.v[x] = d + x < a.hd ? from[min(x, a.hd - 1 - d)] : (T)0.0f;
        *reinterpret_cast<Pack<T, VEC>*>(kpage + (((unsigned)(h0 + h) << a.pshift) * a.W + (unsigned)(lo_slot + s) * a.W + d)) = out;
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int j = 0; j < OLD; ++j) {
    const int i = tid + 256 * j;
    if (i >= nh * a.hd) break;
    const long long at = (page_head + h0 + i / a.hd) * a.W + i % a.hd;
    ((T*)a.kmin)[at] = (T)(merge ? smaller(s_lo[i], old_lo[j]) : s_lo[i]);
    ((T*)a.kmax)[at] = (T)(merge ? larger(s_hi[i], old_hi[j]) : s_hi[i]);
  }
}

// ---- attention over pages ---------------------------------------------------------------------------------------------------------------
// softmax(q k^T scale) v of the query rows that share a key-value head, over virtual keys i = entry * P + offset: entry e is table slot
// e, or slot selected[e].  A workgroup of 4 waves takes a run of keys of one unit (context, key-value head, 16 RT rows); the waves take
// tiles of 32 keys in turn, each with a running maximum and sum of its own, merged through LDS at the end.  Both products run on the
// matrix cores without a pass through LDS: S^T = K Q^T leaves lane group g of a tile with the scores of its keys, which are the operand
// that O^T = V^T P^T takes from that lane group -- the rows of K are dealt out so that they are 8 neighbouring keys (4 in 32-bit pages), i.e. one
// 16-byte load of a value row.  What bounds it is the single pass over keys and values:
// 240 us for 64 contexts of up to 8191 tokens, 8 heads of 128 shared by 32 (1.2 GB: 5.0 TB/s), 741 us for one of 1 000 003 (4.1 GB: 5.5 TB/s); short
// contexts by the chain length, page, keys, values and the join: 6 + 4 us for 3080 tokens of 8 heads of 15.  A wave asks for a tile, waits and
// works, so a launch of few workgroups waits most of its time: 15.5 us for 56 MB of selected pages (336 workgroups, 32-bit).  A pass serves 32
// query rows of a key-value head (16 of 256 channels): more of them read keys and values again (226 us for 16 tokens, 241 for 32, 318 for 33,
// 32 contexts of up to 20 011 tokens, 12 heads of 64, float16).
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
    u.n = a.count << a.pshift;  // (whatever the length: an empty context's keys are masked)
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
  constexpr int NV = NC * (F32 ? 2 : 1);                          // 16-byte value loads of a tile
  constexpr bool EARLY = NV * RT <= 8;
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
      if (page >= 0 && page < a.num_pages) valid = min(max(max(a.lengths[u.b], 0) - (logical << a.pshift), 0), P);
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
      // the values' loads go out with the keys', where there are registers for both (in 32-bit pages with the first 16 keys'; the other 16
      // are asked for once those are multiplied)
      uint4 early[EARLY ? NV : 1];
      if constexpr (EARLY) {
#pragma unroll
        for (int t = 0; t < (F32 ? 2 : 1); ++t) {
          const int i = base + (F32 ? 16 * t : 8 * g), e = min((i >> a.pshift) - e0, ne - 1);
          const T* vr = values + s_page[e] * page_stride + (long long)r16 * P + (i & (P - 1)) + (F32 ? 4 * g : 0);
#pragma unroll
          for (int c = 0; c < NC; ++c) early[t * NC + c] = *reinterpret_cast<const uint4*>(vr + (long long)16 * c * P);
        }
      }
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
            f32x4 vf = EARLY ? __builtin_bit_cast(f32x4, early[EARLY ? t * NC + c : 0]) : *reinterpret_cast<const f32x4*>(vr + (long long)16 * c * P);
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
          typename Mma<T>::V8 vf = __builtin_bit_cast(typename Mma<T>::V8, EARLY ? early[EARLY ? c : 0] : *reinterpret_cast<const uint4*>(vr + (long long)16 * c * P));
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

// The join of a row's splits.  Up to 64: a wave a row; lane s holds the weight of split s, W / 4 lanes a split's channels.
template <class T, int W>
__global__ __launch_bounds__(256) void k_paged_join(AttArgs a, int rows_per_block, int blocks, int rows) {
  constexpr int L = W == 96 ? 32 : W / 4, N = 64 / L;  // lanes of a split, splits side by side
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= rows) return;
  const int r_in = r % a.rows, unit = r / a.rows * a.row_blocks + r_in / rows_per_block;
  const Unit u = unit_of(a, unit);
  const int chunk = split_chunk(u.n, a.splits);
  if (u.n <= chunk) return;
  const int ns = (u.n + chunk - 1) / chunk;
  const float2* ml = reinterpret_cast<const float2*>(a.part + (long long)blocks * rows_per_block * W);
  const long long first = ((long long)unit * a.splits) * rows_per_block + r_in % rows_per_block;
  const float2 mine = lane < ns ? ml[first + (long long)lane * rows_per_block] : float2{-FLT_MAX, 0.0f};
  float top = mine.x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float f = __builtin_amdgcn_exp2f(mine.x - top);
  float sum = f * mine.y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  const int c = lane % L, n = lane / L;
  f32x4 acc = {0, 0, 0, 0};
  for (int s0 = 0; s0 < ns; s0 += N) {
    const int s = min(s0 + n, ns - 1);
    const float fs = __shfl(f, s), w = s0 + n < ns ? fs : 0.0f;  // (every lane gives its weight, also one whose own turn is over)
    if (W != 96 || c < W / 4) acc += w * *reinterpret_cast<const f32x4*>(a.part + (first + (long long)s * rows_per_block) * W + 4 * c);
  }
#pragma unroll
  for (int d = L; d < 64; d <<= 1)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor(acc[x], d);
  if (n > 0) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T* out = (T*)a.out + row_offset(a, u, r_in);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (4 * c + x < a.hd) out[4 * c + x] = (T)(acc[x] * inv);
}

// More than 64: a workgroup a row; the weights are laid into LDS first, so that the reads of the partial results do not wait for each
// other, and its groups of W / 4 threads take the splits in turn.  Sums in a fixed order in both.
constexpr int kJoinSplits = 512;
template <class T, int W>
__global__ __launch_bounds__(512) void k_paged_join_many(AttArgs a, int rows_per_block, int blocks) {
  constexpr int L = W / 4, N = 512 / L;
  __shared__ f32x4 s_o[N][L];
  __shared__ float s_w[kJoinSplits], s_top[8], s_sum[8];
  const int r_in = blockIdx.x % a.rows, unit = blockIdx.x / a.rows * a.row_blocks + r_in / rows_per_block;
  const Unit u = unit_of(a, unit);
  const int chunk = split_chunk(u.n, a.splits);
  if (u.n <= chunk) return;
  const int ns = (u.n + chunk - 1) / chunk, tid = threadIdx.x;
  const float2* ml = reinterpret_cast<const float2*>(a.part + (long long)blocks * rows_per_block * W);
  const long long first = ((long long)unit * a.splits) * rows_per_block + r_in % rows_per_block;
  const float2 mine = tid < ns ? ml[first + (long long)tid * rows_per_block] : float2{-FLT_MAX, 0.0f};
  float top = mine.x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((tid & 63) == 0) s_top[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, s_top[w]);
  const float f = __builtin_amdgcn_exp2f(mine.x - top);
  s_w[tid] = f;
  float l = f * mine.y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  if ((tid & 63) == 0) s_sum[tid >> 6] = l;
  __syncthreads();
  const int c = tid % L, n = tid / L;
  f32x4 acc = {0, 0, 0, 0};
  if (n < N) {
#pragma unroll 8
    for (int s = n; s < ns; s += N) acc += s_w[s] * *reinterpret_cast<const f32x4*>(a.part + (first + (long long)s * rows_per_block) * W + 4 * c);
    s_o[n][c] = acc;
  }
  __syncthreads();
  if (tid < L) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += s_sum[w];
    f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < N; ++i) v += s_o[i][c];
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
  int segments;    // of a long row
  int* chosen;     // [B, T, H, segments, count]: the best of each
};

// One summary is read once: W / 8 lanes take 8 channels of a page each, 64 / that many pages side by side in a wave, two such sets at a
// time as 64-bit numbers in registers, all query rows over them.  The lanes' sums meet in a rotation within the 16-lane row, whose result
// is the same in every lane.  What bounds it: a step waits for its summaries before its sums begin -- only the table entries of the next are
// fetched ahead --, so read and work add up (31 us for 76 MB, 4 rows of 128 channels; the read alone is 15 us at a copy's rate, the 64-bit
// multiplications 4 at the card's).  Tried and left: the 64-bit matrix instruction (42 TFLOP/s, and it pays for 16 rows whatever their
// number); 32-bit scores of all pages with a bound on their error and 64-bit ones near the border alone (26 us here, but 5 to 7 more in the
// selection, and 7 more where rows are short).
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

constexpr int kScorePages = 2;  // pages of a lane group at a time
constexpr int kQueryRows = 8;   // query rows in LDS

template <class T, int W>
__global__ __launch_bounds__(256) void k_paged_score(SelectArgs a) {
  constexpr int L = W == 96 ? 16 : W / 8, GP = 64 / L, NP = kScorePages, STEP = NP * GP, N = 16 / sizeof(T);
  __shared__ double2 s_q[kQueryRows][8][L];  // {max(q, 0), min(q, 0)} of channel 8 l + j at [row][j][l]
  // (heads next to each other: their summaries of a page are; 31 us against 35 for 16 contexts of up to 2048 pages)
  const int h = blockIdx.x % a.H, block = blockIdx.x / a.H % a.score_blocks, b = blockIdx.x / a.H / a.score_blocks;
  const int P = 1 << a.pshift;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane % L, c0 = lc * 8, gp = lane / L;
  const int per_block = 4 * STEP * a.score_steps;
  const int rows = a.T * a.G;
  // what does not depend on the context's length is asked for before it: the first step's table entries, then the query, whose loads each
  // stand under a condition of their own and wait one for the other (four for heads of 128)
  auto entries = [&](int first, int (&page)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) page[i] = a.table[(long long)b * a.slots + min(first + i * GP + gp, a.slots - 1)];
  };
  constexpr int PER = kQueryRows * 8 * L / 256 > 0 ? kQueryRows * 8 * L / 256 : 1;
  float q0[PER];
  auto query = [&](int r0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i, r = r0 + at / (8 * L), c = at % (8 * L);
      q0[i] = r < rows && c < a.hd ? to_f(((const T*)a.q)[(((long long)b * a.T + r / a.G) * a.heads + (long long)h * a.G + r % a.G) * a.hd + c]) : 0.0f;
    }
  };
  auto lay = [&]() {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + 256 * i, c = at % (8 * L);
      const float x = q0[i];
      if (at < kQueryRows * 8 * L) s_q[at / (8 * L)][c % 8][c / 8] = double2{(double)(x < 0.0f ? 0.0f : x), (double)(x < 0.0f ? x : 0.0f)};  // (a NaN stays)
    }
  };
  int page[NP], next[NP];
  entries(block * per_block + wave * STEP, next);
  query(0);
  const int np = (int)min((long long)a.slots, ((long long)max(a.lengths[b], 0) + P - 1) >> a.pshift);
  if (block * per_block >= np) return;
  lay();
  __syncthreads();
#pragma unroll 1
  for (int step = 0; step < a.score_steps; ++step) {
    const int first = block * per_block + (step * 4 + wave) * STEP;
    if (rows <= kQueryRows && first >= np) break;  // (with more rows the workgroup stays together: it loads them again)
    double mx[NP][8], mn[NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) page[i] = first + i * GP + gp < np && next[i] < a.num_pages ? next[i] : -1;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const long long at = ((long long)max(page[i], 0) * a.H + h) * W + (W == 96 ? min(c0, 88) : c0);
#pragma unroll
      for (int j = 0; j < 8 / N; ++j) {
        const Pack<T, N> hi = reinterpret_cast<const Pack<T, N>*>((const T*)a.kmax + at)[j];
        const Pack<T, N> lo = reinterpret_cast<const Pack<T, N>*>((const T*)a.kmin + at)[j];
#pragma unroll
        for (int x = 0; x < N; ++x) {
          mx[i][N * j + x] = W != 96 || c0 < W ? (double)to_f(hi.v[x]) : 0.0;  // (lanes without channels)
          mn[i][N * j + x] = W != 96 || c0 < W ? (double)to_f(lo.v[x]) : 0.0;
        }
      }
    }
    if (step + 1 < a.score_steps) entries(first + 4 * STEP, next);
    double best[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) best[i] = -INFINITY;
    int g = 0, t = 0;
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      if (rows > kQueryRows && r % kQueryRows == 0) {
        query(r);
        __syncthreads();
        lay();
        __syncthreads();
      }
      double s[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) s[i] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double2 q = s_q[r % kQueryRows][j][lc];
#pragma unroll
        for (int i = 0; i < NP; ++i) s[i] = fma(q.y, mn[i][j], fma(q.x, mx[i][j], s[i]));
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const double x = group_sum<L>(s[i]);
        best[i] = (x > best[i] || x != x) ? x : best[i];
      }
      if (++g == a.G) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int slot = first + i * GP + gp;
          if (slot < np && lc == 0) a.scores[(((long long)b * a.T + t) * a.H + h) * a.slots + slot] = page[i] >= 0 ? best[i] : -INFINITY;
          best[i] = -INFINITY;
        }
        g = 0;
        ++t;
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

// The count best of a row, the lowest slots first among equals, written in ascending order.  The scores are rounded to 32 bits (a monotone
// map: they sort into buckets as the scores do) and their buckets kept in LDS (the part of a row behind CAP pages is read again in each
// pass); the scores themselves are read again only where two of a bucket have to be told apart.  A histogram over equal steps between the
// smallest and the largest finds the bucket that holds the border; up to kFew of a bucket are ranked against each other by score and
// slot.  A bucket with more (many near-equals, or a few scores far from the rest) is divided again by the scores' bits as integers, from
// their highest differing bit: 9 bits a pass and more, so it ends.
// One workgroup a row, and what bounds a long row is what a CU reads and handles: LEVEL 1 takes segments of CAP pages, whose best LEVEL 2
// chooses from (in the slots' order, so equals are told apart as in the row).
constexpr int kFew = 256;
template <int NT, int CAP, int LEVEL>
__global__ __launch_bounds__(NT) void k_paged_select(SelectArgs a) {
  constexpr int NW = NT / 64, NB = 2 * NT, BITS = NT == 1024 ? 11 : 9;
  static_assert(NB == 1 << BITS && kFew <= NT, "two buckets a thread");
  __shared__ int s_bucket[CAP];
  __shared__ int s_hist[NB];
  __shared__ unsigned long long s_lo[NW], s_hi[NW], s_key[kFew], s_last_key;
  __shared__ float s_f[2][NW];
  __shared__ int s_slot[kFew], s_sum[NW], s_bin, s_above, s_few, s_last_slot;
  const long long row = LEVEL == 1 ? blockIdx.x / a.segments : blockIdx.x;
  const int b = (int)(row / ((long long)a.T * a.H)), first = LEVEL == 1 ? (int)(blockIdx.x % a.segments) * CAP : 0;
  const double* __restrict__ sc = a.scores + row * a.slots + first;
  const int* __restrict__ chosen = a.chosen + row * a.segments * a.count;
  int* __restrict__ out = LEVEL == 1 ? a.chosen + (long long)blockIdx.x * a.count : a.out + row * a.count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << a.pshift;
  const int there = (int)min((long long)a.slots, ((long long)max(a.lengths[b], 0) + P - 1) >> a.pshift);
  const int np = LEVEL == 1 ? min(max(there - first, 0), CAP) : LEVEL == 2 ? a.segments * a.count : there;  // entries
  // entry i's slot and score
  auto slot_of = [&](int i) { return LEVEL == 2 ? chosen[i] : first + i; };
  auto score = [&](int i) {
    if constexpr (LEVEL == 2) {
      const int s = chosen[i];
      return s >= 0 ? sc[s] : -(double)INFINITY;
    } else {
      return sc[i];
    }
  };
  // -inf: not there (a score below the range of 32 bits is its lowest value)
  auto rounded = [](double s) { return s == -INFINITY ? -INFINITY : s < -(double)FLT_MAX ? -FLT_MAX : (float)s; };
  const int kept = min(np, CAP);
  constexpr int AT_ONCE = CAP > 4096 ? 16 : 4;
  float flo = INFINITY, fhi = -INFINITY;
  int n = 0;
  auto meet = [&](float x) {
    n += !(x == -INFINITY);
    if (fabsf(x) < INFINITY) {
      flo = fminf(flo, x);
      fhi = fmaxf(fhi, x);
    }
  };
  for (int i0 = tid; i0 < kept; i0 += AT_ONCE * NT) {
    double x[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) x[i] = score(min(i0 + NT * i, np - 1));
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
      if (i0 + NT * i < kept) {
        const float y = rounded(x[i]);
        s_bucket[i0 + NT * i] = __float_as_int(y);
        meet(y);
      }
  }
  for (int i = tid + CAP; i < np; i += NT) meet(rounded(score(i)));
  for (int i = tid; i < NB; i += NT) s_hist[i] = 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    flo = fminf(flo, __shfl_xor(flo, d));
    fhi = fmaxf(fhi, __shfl_xor(fhi, d));
    n += __shfl_xor(n, d);
  }
  if (lane == 0) {
    s_f[0][wave] = flo;
    s_f[1][wave] = fhi;
    s_sum[wave] = n;
  }
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    flo = fminf(flo, s_f[0][w]);
    fhi = fmaxf(fhi, s_f[1][w]);
    n += s_sum[w];
  }
  // The bucket of a score, -1: not there.  (Where the step is infinite or no number -- no two finite scores -- all of them are in bucket 0.)
  const float inv = (float)(NB - 1) / (fhi - flo);
  auto bucket = [&](float x) {  // (branch-free: a row of 31 251 spends its time on these instructions)
    int at = (int)fminf(fmaxf((x - flo) * inv, 0.0f), (float)(NB - 1));
    at = x != x ? NB - 1 : at;
    return x == -INFINITY ? -1 : at;
  };
#pragma unroll 4
  for (int i = tid; i < kept; i += NT) {
    const int at = bucket(__int_as_float(s_bucket[i]));
    s_bucket[i] = at;
    if (at >= 0) atomicAdd(&s_hist[at], 1);
  }
  for (int i = tid + CAP; i < np; i += NT) {
    const int at = bucket(rounded(score(i)));
    if (at >= 0) atomicAdd(&s_hist[at], 1);
  }
  __syncthreads();  // (from here on a wave reads buckets that others wrote, also where the border below is not looked for)
  // buckets above `border` are taken, and of those in it what is above last_key, or equal to it with a slot up to last_slot
  int border = -1, last_slot = 0x7fffffff;
  unsigned long long last_key = 0;
  if (n > a.count) {
    int need = a.count;
    unsigned long long lo = kNotThere + 1, hi = ~0ull;  // keys of the border bucket's candidates
    int shift = -1;
    // f(slot, key) over the candidates
    auto candidates = [&](auto f) {
      auto one = [&](int slot) {
        const unsigned long long k = score_key(score(slot));
        if (k >= lo && k <= hi) f(slot, k);
      };
      for (int i = tid; i < kept; i += NT)
        if (s_bucket[i] == border) one(i);
      for (int i = tid + CAP; i < np; i += NT)
        if (bucket(rounded(score(i))) == border) one(i);
    };
    for (;;) {
      if (tid == 0) s_few = 0;
      __syncthreads();
      // the bucket that holds the border: counts from the top, two buckets a thread
      const int b1 = NB - 1 - 2 * tid, h1 = s_hist[b1], h0 = s_hist[b1 - 1];
      int upto = h1 + h0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      if (lane == 63) s_sum[wave] = upto;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) upto += w < wave ? s_sum[w] : 0;
      const int before = upto - h1 - h0;
      if (before < need && upto >= need) {
        const bool upper = before + h1 >= need;
        s_bin = upper ? b1 : b1 - 1;
        s_above = upper ? before : before + h1;
      }
      __syncthreads();
      const int bin = s_bin, inside = s_hist[bin];
      need -= s_above;
      if (shift < 0) {
        border = bin;
      } else {
        const unsigned long long from = lo + ((unsigned long long)bin << shift);
        const unsigned long long rest = (1ull << shift) - 1;  // (from + rest may pass 2^64: hi is the key of a NaN)
        hi = hi - from > rest ? from + rest : hi;
        lo = from;
      }
      if (inside <= kFew) {
        candidates([&](int slot, unsigned long long k) {
          const int at = atomicAdd(&s_few, 1);  // (any order: the ranks are of key and slot)
          s_key[at] = k;
          s_slot[at] = slot;
        });
        __syncthreads();
        if (tid < inside) {
          const unsigned long long k = s_key[tid];
          const int slot = s_slot[tid];
          int rank = 1;
          for (int i = 0; i < inside; ++i) rank += s_key[i] > k || (s_key[i] == k && s_slot[i] < slot);
          if (rank == need) {
            s_last_key = k;
            s_last_slot = slot;
          }
        }
        __syncthreads();
        last_key = s_last_key;
        last_slot = s_last_slot;
        break;
      }
      // the candidates' smallest and largest key
      unsigned long long bl = ~0ull, bh = 0;
      candidates([&](int, unsigned long long k) {
        bl = min(bl, k);
        bh = max(bh, k);
      });
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        bl = min(bl, (unsigned long long)__shfl_xor((long long)bl, d));
        bh = max(bh, (unsigned long long)__shfl_xor((long long)bh, d));
      }
      if (lane == 0) {
        s_lo[wave] = bl;
        s_hi[wave] = bh;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        bl = min(bl, s_lo[w]);
        bh = max(bh, s_hi[w]);
      }
      lo = bl;
      hi = bh;
      if (lo == hi) {  // many equals: the slot of the need-th of them
        int base = 0;
        for (int i0 = 0; i0 < np && base < need; i0 += NT) {
          const int slot = i0 + tid;
          const bool is = slot < np && score_key(score(slot)) == lo;
          const unsigned long long m = __ballot(is);
          __syncthreads();
          if (lane == 0) s_sum[wave] = __popcll(m);
          __syncthreads();
          int at = base;
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            at += w < wave ? s_sum[w] : 0;
            base += s_sum[w];
          }
          at += __popcll(m & ((1ull << lane) - 1));
          if (is && at == need - 1) s_last_slot = slot;
        }
        __syncthreads();
        last_key = lo;
        last_slot = s_last_slot;
        break;
      }
      shift = max(0, 64 - __clzll((long long)(hi - lo)) - BITS);
      for (int i = tid; i < NB; i += NT) s_hist[i] = 0;
      __syncthreads();
      candidates([&](int, unsigned long long k) { atomicAdd(&s_hist[(int)((k - lo) >> shift)], 1); });
    }
  }

  // a wave takes a run of slots: counted, then written behind the waves before it
  auto taken = [&](int slot, int end) {
    const int at = slot < kept ? s_bucket[min(slot, kept - 1)] : slot < end ? bucket(rounded(score(slot))) : -1;
    bool take = at > border && slot < end;
    if (__any(at == border && border >= 0)) {
      const bool tie = at == border && slot < end;
      const unsigned long long k = tie ? score_key(score(slot)) : 0;
      take = take || (tie && (k > last_key || (k == last_key && slot <= last_slot)));
    }
    return __ballot(take);
  };
  const int run = ((np + NW - 1) / NW + 63) & ~63, from = wave * run, to = min(np, from + run);
  int mine = 0;
  for (int i = from; i < to; i += 64) mine += __popcll(taken(i + lane, to));
  __syncthreads();  // (s_sum's last readers)
  if (lane == 0) s_sum[wave] = mine;
  __syncthreads();
  int base = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    before += w < wave ? s_sum[w] : 0;
    base += s_sum[w];
  }
  if (mine > 0) {
    for (int i = from; i < to; i += 64) {
      const unsigned long long m = taken(i + lane, to);
      const int at = before + __popcll(m & ((1ull << lane) - 1));
      if ((m >> lane & 1) && at < a.count) out[at] = slot_of(i + lane);
      before += __popcll(m);
    }
  }
  for (int i = base + tid; i < a.count; i += NT) out[i] = -1;
}

constexpr long long kMaxThreads = 0xffffffffLL;  // of a grid's dimension

template <class TI, class T>
int append_typed(AppendArgs& a, int units, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);  // 16-byte stores both ways
  // wide loads need whole chunks in a workgroup's heads, every chunk of the row at a multiple of its size, and rotation pairs that start at even channels of the row
  const uintptr_t align = sizeof(TI) * VEC;
  const bool whole = a.hd % VEC == 0;
  const int most = whole ? kAppendRow<2> : kAppendRow<1>;
  const bool wide = VEC / std::gcd(a.hd, VEC) * a.hd <= most && (a.H * a.hd) % VEC == 0 && a.k_stride % VEC == 0 && a.v_stride % VEC == 0 && (uintptr_t)a.k % align == 0 && (uintptr_t)a.v % align == 0 &&
                    (a.rotary == 0 || a.rotary > a.hd || a.hd % 2 == 0);
  // heads of a workgroup: as many workgroups as keep the chip busy, but not fewer than 128 chunks each (of a context's mean number of
  // tokens); whole chunks, not more channels than its tables hold
  const int step = wide ? VEC : 1, unit = step / std::gcd(a.hd, step);
  const int groups = std::max(1, std::min(a.n_tokens / a.B, 1 << a.pshift) / VEC);
  const long long chunks = (long long)a.H * a.hd / step * groups;
  const int parts = (int)std::max(1LL, std::min<long long>({a.H, 2048 / units, chunks / 128}));
  // (a tile of 16 KB: 64 tokens of 64 32-bit channels, 128 of 16 bits)
  const int channels = wide ? (whole ? most : 64 * VEC / 4) : kAppendRow<0>;
  a.heads_per_wg = std::min((a.H + parts - 1) / parts, std::max(1, channels / a.hd));
  a.heads_per_wg = std::max(a.heads_per_wg / unit, 1) * unit;
  const dim3 grid(units, (a.H + a.heads_per_wg - 1) / a.heads_per_wg);
  if (units * 256LL > kMaxThreads || grid.y > 65535) return 2;
  if (wide && whole) k_paged_append<TI, T, 2><<<grid, 256, 0, s>>>(a);
  else if (wide) k_paged_append<TI, T, 1><<<grid, 256, 0, s>>>(a);
  else k_paged_append<TI, T, 0><<<grid, 256, 0, s>>>(a);
  return 0;
}

template <class T, int W, int RT>
void attention_go(const AttArgs& a, int blocks, hipStream_t s) {
  k_paged_attention<T, W, RT><<<blocks, 256, 0, s>>>(a);
  if (a.splits > 1) {
    const int rows = blocks / a.splits / a.row_blocks * a.rows;
    if (a.splits <= 64) k_paged_join<T, W><<<(rows + 3) / 4, 256, 0, s>>>(a, 16 * RT, blocks, rows);
    else k_paged_join_many<T, W><<<rows, 512, 0, s>>>(a, 16 * RT, blocks);
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
// Workgroups for 256 CUs: a unit's keys are split until there are about 2048 (contexts are of unlike length: small pieces even that out;
// 1024 took 291 us for 64 contexts of up to 8191 tokens, 2048 274, 4096 283), or 512 over selected pages, which are as many for each (119
// against 112 us for 16 contexts x 64 pages of 64).  Up to 1024 keys are not split: the join costs what the split saves.
constexpr int kTargetWgs = 2048, kTargetSelected = 512, kAlone = 1024;
AttPlan attention_plan(int B, int T, int H, int G, int W, long long capacity, bool selected) {
  AttPlan p;
  const int rows = selected ? G : T * G;
  p.RT = row_tiles(rows, W);
  p.row_blocks = (rows + 16 * p.RT - 1) / (16 * p.RT);
  p.units = (long long)B * (selected ? T : 1) * H * p.row_blocks;
  const long long most = capacity <= kAlone ? 1 : (capacity + kMinChunk - 1) / kMinChunk;
  p.splits = (int)std::min({most, (long long)kJoinSplits, std::max(1LL, (selected ? kTargetSelected : kTargetWgs) / std::max(1LL, p.units))});
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
  if (type == 0 && in_type == 0) return append_typed<float, float>(a, units, s);
  if (type == 1 && in_type == 0) return append_typed<float, _Float16>(a, units, s);
  if (type == 2 && in_type == 0) return append_typed<float, __bf16>(a, units, s);
  if (type == 1 && in_type == 1) return append_typed<_Float16, _Float16>(a, units, s);
  if (type == 2 && in_type == 2) return append_typed<__bf16, __bf16>(a, units, s);
  return 1;
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
  // (the join's rows are at most 32 times the units, 64 threads each)
  if (p.units * p.splits * 256 > kMaxThreads || p.units * 32 * 64 > kMaxThreads) return 2;
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

constexpr int kShortRow = 1536, kSegment = 4096;
// the scores, and for rows of several segments the best of each (at most kSegment slots in all)
long long paged_select_workspace_doubles(int B, int T, int H, int slots) {
  return (long long)B * T * H * (slots + (slots > 2 * kSegment ? kSegment / 2 : 0));
}

int launch_paged_select(const void* q, const void* kmin, const void* kmax, int type, const int* table, const int* lengths, int B, int T, int H, int G,
                        int hd, int slots, int num_pages, int pshift, int count, double* work, int* out, hipStream_t s) {
  if ((long long)B * T * H * 1024 * (slots > 2 * kSegment ? (slots + kSegment - 1) / kSegment : 1) > kMaxThreads || (long long)T * G > 0x7fffffffLL) return 2;
  SelectArgs a{};
  a.q = q, a.kmin = kmin, a.kmax = kmax, a.table = table, a.lengths = lengths;
  a.B = B, a.T = T, a.heads = H * G, a.H = H, a.G = G, a.hd = hd, a.W = paged_width(hd), a.slots = slots, a.num_pages = num_pages, a.pshift = pshift;
  a.count = count, a.scores = work, a.out = out;
  a.segments = (slots + kSegment - 1) / kSegment, a.chosen = (int*)(work + (long long)B * T * H * slots);
  const int L = a.W == 96 ? 16 : a.W / 8, per_step = 4 * kScorePages * (64 / L);  // pages of a workgroup's step
  const long long all_steps = (long long)B * H * ((slots + per_step - 1) / per_step);
  a.score_steps = (int)std::min(16LL, std::max(1LL, all_steps / 2048));  // about 8 workgroups a CU, each with its query loaded once
  a.score_blocks = (slots + per_step * a.score_steps - 1) / (per_step * a.score_steps);
  if ((long long)B * H * a.score_blocks * 256 > kMaxThreads) return 2;
  const int blocks = B * H * a.score_blocks;
  if (type == 0) score_typed<float>(a, blocks, s);
  else if (type == 1) score_typed<_Float16>(a, blocks, s);
  else score_typed<__bf16>(a, blocks, s);
  // Short rows take four waves, where barriers are the time (336 rows of 1251 pages: 8.8 us, 12 with sixteen waves; 128 rows of up to 2048:
  // 10.3 against 8.6).  Rows that a workgroup takes long over are cut into segments where the segments' best are few (31 251 pages, 128 of
  // them: 18 us in two launches, 29 in one).
  const int rows = B * T * H;
  if (slots <= kShortRow) {
    k_paged_select<256, kShortRow, 0><<<rows, 256, 0, s>>>(a);
  } else if (slots <= 2 * kSegment) {
    k_paged_select<1024, 2 * kSegment, 0><<<rows, 1024, 0, s>>>(a);
  } else if ((long long)a.segments * count <= kSegment) {
    k_paged_select<1024, kSegment, 1><<<rows * a.segments, 1024, 0, s>>>(a);
    k_paged_select<1024, kSegment, 2><<<rows, 1024, 0, s>>>(a);
  } else {
    k_paged_select<1024, 32768, 0><<<rows, 1024, 0, s>>>(a);
  }
  return 0;
}

}  // namespace mmf
