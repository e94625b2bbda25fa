// Attention with a learned relative position bias (gfx950), head size 64 or 128.
//
//   s_ij = scale <q_i, k_j> + beta_h(j - i),  beta_h(d) = table[map[clamp(d)]][h]
//   P = softmax_j(s) over the keys allowed by the key mask (and j <= i),
//   O = P V; a row with no key allowed is zero.
//   dV = P^T dO, dP = dO V^T, D_i = <dO_i, O_i>, dS = P (dP - D),
//   dQ = scale dS K, dK = scale dS^T Q, dtable[n][h] = sum of dS where map = n
//
// Layout. v_mfma_f32_32x32x16_bf16: A[m][k] has m = lane & 31, k = 8 (lane >> 5)
// + e; B[k][n] likewise; C has column lane & 31 and row (r & 3) + 8 (r >> 2) +
// 4 (lane >> 5). Every product is written so that the axis that a softmax row
// or a gradient row belongs to is the C column: a lane then owns a whole query
// (or key), its maximum and sum are registers, and the one cross-lane step is
// between the two halves of the wave. The second product contracts over C's
// rows: its B operand is C itself, rounded, with the rows in the order that the
// registers hold them, and its A operand is read from LDS in that same order by
// the transposing 64-bit read (each lane gets four rows of one column). So no
// tile is ever exchanged between lanes or written back.
//
// The bias enters as C's initial value (beta / scale), so it costs no addition:
// where all of a 32x32 tile is further than the largest distance it is one
// constant, else four neighbouring offsets come as one 16-byte LDS read from a
// table kept in four copies, each shifted by one entry, so that every start is
// aligned.
//
// 32 bits: scores, maxima, sums, D, dS for the table's gradient, accumulators.
// Rounded to bf16: P and dS before the second product (a relative 2^-9 of each,
// which the matrix instruction's operands force), and the outputs.
//
// Times at each kernel are medians of 200 passes under the profiler on one
// MI355X of two workloads: "padded", 16x512 with lengths of all sizes, 12 heads,
// D 64; "long", 2x4093 causal, 16 heads over 4, D 128. (The first 20 passes
// of the long case took 173, 267 and 341 us there.) The forward and both backward kernels are bound by the
// vector unit beside the matrix unit: a 32x32 tile takes 8 matrix instructions at
// D 64 in the forward and some 90 vector ones (16 exponentials at a quarter of
// the rate), and two waves of a SIMD overlap them little (16 matrix instructions
// alone 458 ns, 128 vector ones 470, both by turns 749). Without a mask or the
// causal order (8x4096, 16 heads, D 128) the three run at 75 to 80 % of the rate
// of a large library product.

#include <hip/hip_runtime.h>

#include "ga_ops.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 b8;
typedef __attribute__((ext_vector_type(4))) __bf16 b4;
typedef __attribute__((ext_vector_type(4))) short s4;
typedef __attribute__((ext_vector_type(8))) short s8;
typedef __attribute__((ext_vector_type(2))) float f2;
typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(16))) float f16;
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(3))) char lds_char;

#define LOG2E 1.44269504088896340736f
#define INF __builtin_inff()

constexpr int KC = 64;     // rows of a staged chunk
constexpr float LARGE = 4096.f;  // of a row's maximum: from here on half its last bit is 2^-12, a relative 2^-12.5 of P
constexpr int TILE = GA_REL_TILE;  // rows of a workgroup: four waves of 32

// ---- LDS tiles: [rows][D] bf16, 16-byte pieces XORed by a function of the row.
// LDS serves 256 bytes at a time: sixteen neighbouring rows' pieces at one
// column (row reads), or 64 bytes of each of four neighbouring rows (the
// transposing reads); the function sends both to 256 bytes of different banks
// (a row of D = 64 is half of them, and which half is its lowest bit). So the
// tiles' reads do not conflict; those of the bias do, see bias_tile.
template <int D>
__device__ __forceinline__ int piece(int row, int p) {
  const int f = D == 64 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
  return row * 2 * D + ((p ^ f) << 4);
}

// A fragment, rows of the tile as m: row `row`, columns 16 t + 8 hi ..
template <int D>
__device__ __forceinline__ b8 row_frag(const char* tile, int row, int t, int hi) {
  return *(const b8*)(tile + piece<D>(row, 2 * t + hi));
}

// A fragment, columns of the tile as m (32 dt ..), 16 rows from `row` as k in
// the order of C's registers
template <int D>
__device__ __forceinline__ b8 col_frag(const char* tile, int row, int dt, int lane) {
  const int t = lane & 15, r = row + 4 * (lane >> 5) + (t >> 2);
  const int p = 4 * dt + 2 * ((lane >> 4) & 1) + ((t & 3) >> 1);
  const int in = (t & 1) << 3;
  const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(tile + piece<D>(r, p) + in));
  const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(tile + piece<D>(r + 8, p) + in));
  return __builtin_bit_cast(b8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// order of the instructions around: four LDS reads, then one for each matrix
// instruction, so that a read's latency lies behind the products before it
template <int N>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
  for (int i = 0; i < N - 4; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
}

__device__ __forceinline__ f16 mfma(b8 a, b8 b, f16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// one instruction of three operands, and a NaN stays
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ int crow(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }

// C's registers 8 ks .. 8 ks + 7 as the B fragment of k-step ks
__device__ __forceinline__ b8 pack(const f16& c, int ks) {
  b8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (__bf16)c[8 * ks + e];
  return v;
}

// ---- staging of 64 rows of two matrices by T threads, straight from memory
// into LDS (16 bytes a lane, a wave's 1 KB side by side), so that no register
// waits for a load: the next chunk arrives while this one is computed. The
// tile's order is made by the addresses that the lanes read. Issued by inline
// assembly, because behind the builtin the compiler waits for the data before
// any LDS read that follows; the instruction has no register result. m0 is
// reserved, so the compiler takes no clobber of it: in the code that it makes of
// these kernels no other instruction names m0. After `wait`, `clear` zeroes the rows
// that must not count (masked keys, rows past the end): what stands there, NaN
// too, cannot reach a result. Ordinary loads of the loop are issued before the
// chunk's and used after `wait`, or their own wait would be for the chunk too.
template <int D, int T = 256>
struct Stage {
  static constexpr int N = KC * D / 8 / T;  // pieces a thread, each matrix
  unsigned ax[N], ay[N];                      // byte offsets inside a chunk

  __device__ __forceinline__ static int place(int i) { return (threadIdx.x + T * i) * 16; }  // in a tile
  __device__ __forceinline__ static int row(int i) { return place(i) / (2 * D); }
  // the piece that lies there: piece() is its own inverse
  __device__ __forceinline__ static int col(int i) { return (piece<D>(row(i), place(i) / 16 % (D / 8)) - row(i) * 2 * D) / 2; }

  __device__ __forceinline__ void init(int sx, int sy) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      ax[i] = 2u * (row(i) * sx + col(i));
      ay[i] = 2u * (row(i) * sy + col(i));
    }
  }
  __device__ __forceinline__ static void move(const char* from, unsigned at, unsigned to) {
    extern __shared__ __align__(16) char smem[];
    const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_char*)smem + to);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(at), "s"(from) : "memory");
  }
  // rows r0 .. r0 + 63 of matrices with row strides sx, sy to tiles tx, ty bytes behind the kernel's LDS; rows from
  // `end` on repeat the last one
  __device__ __forceinline__ void load(const __bf16* px, int sx, const __bf16* py, int sy, int r0, int end, unsigned tx, unsigned ty) {
    const char* bx = (const char*)(px + (long long)r0 * sx);
    const char* by = (const char*)(py + (long long)r0 * sy);
    const int wave = (threadIdx.x >> 6) * 1024;
    const bool whole = r0 + KC <= end;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned x = ax[i], y = ay[i];
      if (!whole) {
        const int r = min(row(i), end - 1 - r0);
        x = 2u * (r * sx + col(i));
        y = 2u * (r * sy + col(i));
      }
      move(bx, x, tx + wave + 16 * T * i);
      move(by, y, ty + wave + 16 * T * i);
    }
  }
  __device__ __forceinline__ static void wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0); the compiler knows it, and waits for no earlier load again
    asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ void scale(char* ty, const float* by, int r0, int end) {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      b8* p = (b8*)(ty + place(i));
      const float f = by[min(r0 + row(i), end - 1)];
      b8 v = *p;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (__bf16)((float)v[e] * f);
      *p = v;
    }
  }
  __device__ __forceinline__ void clear(char* tx, char* ty, unsigned long long on) {
    if (on != ~0ull) {
      const b8 zero = {};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!((on >> row(i)) & 1)) {
          *(b8*)(tx + place(i)) = zero;
          *(b8*)(ty + place(i)) = zero;
        }
    }
  }
};

// ---- the bias of one head in LDS: entry x is the offset clamp(x - 7 - far),
// copy c holds the entries from c on.
__host__ __device__ __forceinline__ int bias_top(int far) { return (2 * far + 10) & ~3; }  // from here on all are the last offset's
__host__ __device__ __forceinline__ int bias_len(int far) { return bias_top(far) + 4; }

// Table values from -2^29 down (-1e9, the type's lowest) stand for a mask, as
// -inf does: divided by the scale the lowest would leave 32 bits' range.
__device__ __forceinline__ float as_bias(__bf16 t, float scale) {
  const float f = (float)t;
  return f <= -536870912.f ? -INF : f / scale;
}

// a value that all lanes share, where a scalar register can hold it
__device__ __forceinline__ float shared(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// A bias beyond the largest distance in the exponent, in base 2, and what that
// product's rounding left out: with large values it would outweigh the scores.
struct Flat {
  float hi, lo;
  __device__ __forceinline__ Flat(float bias, float c2) : hi(shared(bias * c2)), lo(shared(fabsf(hi) < INF ? fmaf(bias, c2, -hi) : 0.f)) {}
};

__device__ __forceinline__ void put_bias(float* bias, int len, int x, float v) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (x >= c && x - c < len) bias[c * len + x - c] = v;
}

// In two steps, so that the two dependent loads of an entry run beside the
// kernel's other first loads: the constructor issues them, `put` stores. T threads;
// mirrored: the offset of an entry with its sign turned.
template <int T = 256, bool MIRRORED = false>
struct Bias {
  static constexpr int N = (2 * GA_REL_MAX_DISTANCE + 17 + T - 1) / T;
  __bf16 t[N];
  int len;
  __device__ __forceinline__ Bias(const RelArgs& a, int h) : len(bias_len(a.far)) {
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * T >= len + 3) break;
      const int d = min(max((int)threadIdx.x + T * i - 7 - a.far, -a.far), a.far);
      n[i] = a.map[(MIRRORED ? -d : d) + a.far];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * T >= len + 3) break;
      t[i] = a.table[(long long)min(max(n[i], 0), a.buckets - 1) * a.NH + h];
    }
  }
  __device__ __forceinline__ void put(float scale, float* bias) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * T >= len + 3) break;
      put_bias(bias, len, threadIdx.x + T * i, as_bias(t[i], scale));
    }
  }
};

// C's initial value for rows u0 + crow(r) against column w: the bias of the
// offset row - column. `low`, `high`: the values beyond the largest distance.
// The four copies lie bias_len floats apart, 12 modulo the 64 banks at distances
// 64, 128, 256 and 512: the sixteen lanes of a read touch 13 different places of
// 16 bytes instead of 16, so it takes twice its time. That is what the counters
// show as conflicts: 27, 19 and 17 % of the LDS cycles of the three kernels on
// "padded", 5, 4 and 2 % on "long".
__device__ __forceinline__ f16 bias_tile(const float* bias, int far, int row0, int col0, int lane, float low, float high) {
  f16 c;
  if (row0 + 31 - col0 <= -far || row0 - (col0 + 31) >= far) {
    const float v = row0 < col0 ? low : high;
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = v;
    return c;
  }
  // which copy is the lane's own, since tiles start on multiples of 32
  const int x = row0 + 4 * (lane >> 5) - (col0 + (lane & 31)) + far + 7, copy = x & 3;
  const float* mine = bias + copy * bias_len(far);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f4 v = *(const f4*)(mine + min(max((x & ~3) + 8 * g, 0), bias_top(far)));
#pragma unroll
    for (int e = 0; e < 4; ++e) c[4 * g + e] = v[e];
  }
  return c;
}

// Which tile of which head a workgroup works on. Workgroups go to the eight XCDs
// by turns, and each XCD has an L2 of its own, so all tiles of the heads that
// share keys go to one XCD; neighbouring units (a batch's key heads) go to
// different ones, since batches differ in length. Under the causal mask tiles
// differ in work too (and key tiles of a padded batch do): of some 64 workgroups at a time the longest start first.
// `units` share nothing with each other, `per` columns of a unit share its keys
// (query heads, or parts of them). Returns unit * per + column.
__device__ __forceinline__ int place(int at, int units, int per, int tiles, bool by_work, int& tile) {
  int xcd = 0, step = 1, columns = units * per;
  if ((units & 7) == 0) {
    xcd = at & 7;
    at >>= 3;
    step = 8;
    columns >>= 3;
  }
  int c;
  if (by_work) {
    const int most = max(1, 64 / tiles), first = at / (most * tiles) * most, n = min(most, columns - first);
    at -= first * tiles;
    tile = at / n;
    c = first + at % n;
  } else {
    tile = at % tiles;
    c = at / tiles;
  }
  return (xcd + c / per * step) * per + c % per;
}

// one past the last key that the mask leaves, 0 if it leaves none. All threads.
__device__ int mask_end(const unsigned char* mask, int end, int* lds) {
  int last = 0;
  for (int j = threadIdx.x; j < end; j += 256)
    if (mask[j]) last = j + 1;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = last;
  __syncthreads();
  last = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
  return last;
}

// this lane's mask byte of a chunk of 64 keys
__device__ __forceinline__ int key_byte(const unsigned char* mask, int j0, int end) {
  return mask ? mask[min(j0 + (int)(threadIdx.x & 63), end - 1)] : 1;
}

// C rows whose key does not count, or lies behind the column's query -> fill
__device__ __forceinline__ void drop_rows(f16& c, unsigned bits, bool diag, int key0, int query0, int lane, float fill) {
  // the empty statements keep these branches: as selects they would run in every tile
  const int hi = lane >> 5;
  if (bits != ~0u) {
    asm volatile("");
    const unsigned b = bits >> (4 * hi);
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = (b >> crow(r, 0)) & 1 ? c[r] : fill;
  }
  if (diag) {
    asm volatile("");
    const int most = query0 + (lane & 31) - key0 - 4 * hi;
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = crow(r, 0) <= most ? c[r] : fill;
  }
}

template <int D>
__device__ __forceinline__ void store_columns(float* row, const f16* c, float mul, int hi) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = c[dt][4 * g + e] * mul;
      *(f4*)(row + 32 * dt + 8 * g + 4 * hi) = v;
    }
}

// The wave's 32 columns of C as bf16 rows of memory, `count` of them, by way of its
// own 64 D bytes of LDS: whole rows, 16 bytes a lane. From the registers every store
// would touch 32 rows with 16 bytes each: dK and dV took 54 us instead of 47.5 at
// 16x512 padded, 8 heads, D 128. The fp32 parts gained nothing by it.
template <int D>
__device__ __forceinline__ void store_rows(char* tile, __bf16* to, long long stride, int count, const f16* c, float mul, int lane) {
  const int hi = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      b4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (__bf16)(c[dt][4 * g + e] * mul);
      *(b4*)(tile + piece<D>(lane & 31, 4 * dt + g) + 8 * hi) = v;
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    const int r = (lane + 64 * n) / (D / 8), p = lane % (D / 8);
    const b8 v = *(const b8*)(tile + piece<D>(r, p));
    if (r < count) *(b8*)(to + r * stride + 8 * p) = v;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// P = exp2(s - lse) * rest. A large maximum (a large bias that all keys of the row
// share) has no bits left for the sum's logarithm: the sum stays apart.
__device__ __forceinline__ void save_lse(float* lse, long long rows, float m, float l) {
  const bool apart = fabsf(m) >= LARGE && l != 0.f;
  lse[0] = l == 0.f ? INF : apart ? m : m + __builtin_amdgcn_logf(l);
  lse[rows] = apart ? 1.f / l : 1.f;
}

// ---------------- forward: a wave owns 32 queries, chunks of 64 keys ----------------
// padded 23 us (matrix unit 22 % busy), long 160 us (47 %, 859 TFLOP/s)
template <int D>
__global__ __launch_bounds__(256, 2) void k_rel_fwd(RelArgs a, int tiles) {
  extern __shared__ __align__(16) char smem[];  // the tiles lie in the first 64 KB, which m0 reaches
  char* buf = smem;  // [2][K, V]
  constexpr int MAT = KC * 2 * D;
  float* bias = (float*)(smem + 4 * MAT);
  int* ends = (int*)(bias + 4 * bias_len(a.far));

  int tile;
  const int column = place(blockIdx.x, a.B * a.NKV, a.NH / a.NKV * a.spans, tiles, a.causal, tile);
  const int bh = column / a.spans, span = column % a.spans;  // a span of the keys
  const int h = bh % a.NH, b = bh / a.NH, hk = h / (a.NH / a.NKV);
  if (a.causal) tile = tiles - 1 - tile;  // the last tile has the most keys
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int i0 = tile * TILE + (threadIdx.x >> 6) * 32, i = i0 + (lane & 31);
  const __bf16* k = a.qkv + (long long)b * a.S * a.width + (a.NH + hk) * D;
  const __bf16* v = k + a.NKV * D;
  const unsigned char* mask = a.mask ? a.mask + (long long)b * a.S : nullptr;

  int end = a.causal ? min(a.S, tile * TILE + TILE) : a.S;  // shorter once the mask is read

  Stage<D> st;
  st.init(a.width, a.width);
  unsigned long long bits = 0, next = 0;
  int key = 0;
  auto fetch = [&](int c) {
    const unsigned to = (c & 1) * 2 * MAT;
    key = key_byte(mask, c * KC, end);
    st.load(k, a.width, v, a.width, c * KC, end, to, to + MAT);
  };
  auto arrive = [&](int c) {
    char* to = buf + (c & 1) * 2 * MAT;
    st.wait();
    next = __ballot(c * KC + lane < end && key != 0);
    st.clear(to, to + MAT, next);
  };
  // everything that the first chunk needs is on its way at once
  const int all = (end + KC - 1) / KC, first = __builtin_amdgcn_readfirstlane(all * span / a.spans);
  fetch(first);
  const Bias<> first_bias(a, h);
  if (mask) end = mask_end(mask, end, ends);
  const int chunks = min((end + KC - 1) / KC, all * (span + 1) / a.spans);
  b8 q[D / 16];
  const __bf16* qp = a.qkv + ((long long)b * a.S + min(i, a.S - 1)) * a.width + h * D;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) q[t] = *(const b8*)(qp + 16 * t + 8 * hi);
  first_bias.put(a.scale, bias);
  st.wait();
  if (first < chunks) arrive(first);
  __syncthreads();

  f16 o[D / 32] = {};
  float m = -INF, l = 0.f;
  const float c2 = a.scale * LOG2E;
  const float low = shared(bias[0]), high = shared(bias[2 * a.far + 7]);
  const Flat flat_low(low, c2), flat_high(high, c2);

  for (int c = first; c < chunks; ++c) {
    bits = next;
    if (c > first) __syncthreads();
    if (c + 1 < chunks) fetch(c + 1);
    const char* kt = buf + (c & 1) * 2 * MAT;
    const char* vt = kt + MAT;
    const int j0 = c * KC;
    if (bits != 0 && !(a.causal && j0 > i0 + 31)) {
      f16 s[2];
      // where all 64 keys lie beyond the largest distance the bias goes into the
      // exponent, and the products start from zero: 32 moves less
      float flat = 0.f, flat_lo = 0.f;
      if (j0 + 63 - i0 <= -a.far || j0 - (i0 + 31) >= a.far) {
        flat = j0 < i0 ? flat_low.hi : flat_high.hi;
        flat_lo = j0 < i0 ? flat_low.lo : flat_high.lo;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) s[sub] = mfma(row_frag<D>(kt, 32 * sub + (lane & 31), 0, hi), q[0], (f16){});
#pragma unroll
        for (int t = 1; t < D / 16; ++t)
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) s[sub] = mfma(row_frag<D>(kt, 32 * sub + (lane & 31), t, hi), q[t], s[sub]);
        reads_ahead<D / 8>();
      } else {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) s[sub] = bias_tile(bias, a.far, j0 + 32 * sub, i0, lane, low, high);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) s[sub] = mfma(row_frag<D>(kt, 32 * sub + (lane & 31), t, hi), q[t], s[sub]);
        reads_ahead<D / 8>();
      }
      if (bits != ~0ull || (a.causal && j0 + 63 > i0))
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
          drop_rows(s[sub], (unsigned)(bits >> (32 * sub)), a.causal && j0 + 32 * sub + 31 > i0, j0 + 32 * sub, i0, lane, -INF);
      float top = larger(s[0][0], s[1][0]);
#pragma unroll
      for (int r = 1; r < 16; ++r) top = larger(larger(top, s[0][r]), s[1][r]);
      top = fmaf(top, c2, flat);
      // the maximum moves only where it grew by more than 8 (a factor of 256,
      // far inside 32 bits and the same relative rounding in bf16): after the
      // first chunks the accumulators are hardly ever rescaled, and the two
      // halves of the wave compare their maxima only then
      if (__any(top > m + 8.f)) {
        const float n = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
        const float f = n == -INF ? 1.f : __builtin_amdgcn_exp2f(m - n);
        m = n;
        l *= f;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= f;
      }
      const float base = flat - (m == -INF ? 0.f : m) + flat_lo;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[sub][r] = __builtin_amdgcn_exp2f(fmaf(s[sub][r], c2, base));
          sum += s[sub][r];
        }
        l += sum;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const b8 p = pack(s[sub], ks);
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) o[dt] = mfma(col_frag<D>(vt, 32 * sub + 16 * ks, dt, lane), p, o[dt]);
        }
      }
    }
    if (c + 1 < chunks) arrive(c + 1);
  }
  l += __shfl_xor(l, 32, 64);
  if (a.spans > 1) {
    if (i >= a.S) return;
    const long long rows = (long long)a.B * a.NH * a.S, row = span * rows + (long long)bh * a.S + i;
    store_columns<D>(a.split + row * D, o, 1.f, hi);
    if (hi == 0) *(f2*)(a.split + a.spans * rows * D + row * 2) = f2{m, l};
    return;
  }
  __syncthreads();  // the tiles are read
  store_rows<D>(smem + (threadIdx.x >> 6) * 64 * D, a.out + (((long long)b * a.S + i0) * a.NH + h) * D, a.NH * D, a.S - i0, o,
                l == 0.f ? 0.f : 1.f / l, lane);
  if (i < a.S && a.lse && hi == 0) save_lse(a.lse + (long long)bh * a.S + i, (long long)a.B * a.NH * a.S, m, l);
}

// joins the spans of a row, in order: four columns a thread (4 to 6 us at up to 32768 rows)
template <int D>
__global__ __launch_bounds__(256) void k_rel_out(RelArgs a) {
  const long long rows = (long long)a.B * a.NH * a.S, row = (long long)blockIdx.x * (1024 / D) + threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  if (row >= rows) return;
  const float* ml = a.split + a.spans * rows * D;
  float m = -INF, l = 0.f;
  for (int s = 0; s < a.spans; ++s) m = larger(m, ml[(s * rows + row) * 2]);
  const float base = m == -INF ? 0.f : m;
  f4 o = {};
  for (int s = 0; s < a.spans; ++s) {
    const f2 x = *(const f2*)(ml + (s * rows + row) * 2);
    const float f = __builtin_amdgcn_exp2f(x[0] - base);
    l = fmaf(x[1], f, l);
    o += *(const f4*)(a.split + (s * rows + row) * D + d) * f;
  }
  const int i = (int)(row % a.S), h = (int)(row / a.S % a.NH);
  const long long b = row / a.S / a.NH;
  const float f = l == 0.f ? 0.f : 1.f / l;
  b4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (__bf16)(o[e] * f);
  *(b4*)(a.out + ((b * a.S + i) * a.NH + h) * D + d) = v;
  if (a.lse && d == 0) save_lse(a.lse + row, rows, m, l);
}

// lane i of each 16 takes lane i + N's value (N < 0: i - |N|), zero from outside
template <int N>
__device__ __forceinline__ float from_lane(float x) {
  if (N == 0) return x;
  constexpr int how = N > 0 ? 0x100 + N : 0x110 - N;
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), how, 0xf, 0xf, true));
}

// Sums of a 32x32 tile along its diagonals. In register r of a lane stands row
// 16 u + s + 4 hi (s = r & 3 | 8 (r >> 2 & 1), u = r >> 3), column 16 ib + i.
// Moved s lanes down within the 16, every register's lane holds the same
// offset but for a multiple of 16, so the additions are plain: d[n] of lane i
// is the sum for the offset first - first column + 4 hi - 16 ib - i + 16 n.
template <int R = 0>
__device__ __forceinline__ void diagonals(const f16& c, float* d) {
  constexpr int s = (R & 3) | ((R & 4) << 1), u = R >> 3;
  d[u] += from_lane<s>(c[R]);
  if (s) d[u + 1] += from_lane<s ? s - 16 : 0>(c[R]);
  if constexpr (R < 15) diagonals<R + 1>(c, d);
}
// ... and the 16 columns of ib = 1 stand 16 offsets lower: with d[1] exchanged
// between the two, d[0] and d[2] are the sums of 32 neighbouring offsets each.
__device__ __forceinline__ void diagonals_32(const f16& c, float* d, bool ib) {
  diagonals(c, d);
  const float other = __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, d[1]), 0x401f));  // lane ^ 16
  d[0] += ib ? 0.f : other;
  d[2] += ib ? other : 0.f;
}

// ---------------- backward 1: dQ, D and the offsets' sums of dS ----------------
// padded 36 us (matrix unit 19 % busy), long 240 us (43 %, 857 TFLOP/s)
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void k_rel_bwd_q(RelArgs a, int tiles) {
  extern __shared__ __align__(16) char smem[];  // the tiles lie in the first 64 KB, which m0 reaches
  char* buf = smem;  // [2][K, V]
  constexpr int MAT = KC * 2 * D;
  float* bias = (float*)(smem + 4 * MAT);
  const int offs = 2 * a.far + 1;
  int* ends = (int*)(bias + 4 * bias_len(a.far));
  float* sums = (float*)(ends + 4);  // [4 waves][2 halves][offs]

  int tile;
  const int column = place(blockIdx.x, a.B * a.NKV, a.NH / a.NKV * a.q_spans, tiles, a.causal, tile);
  const int bh = column / a.q_spans, span = column % a.q_spans;  // a span of the keys
  const int h = bh % a.NH, b = bh / a.NH, hk = h / (a.NH / a.NKV);
  if (a.causal) tile = tiles - 1 - tile;  // the last tile has the most keys
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int i0 = tile * TILE + wave * 32, i = i0 + (lane & 31);
  const __bf16* k = a.qkv + (long long)b * a.S * a.width + (a.NH + hk) * D;
  const __bf16* v = k + a.NKV * D;
  const unsigned char* mask = a.mask ? a.mask + (long long)b * a.S : nullptr;

  int end = a.causal ? min(a.S, tile * TILE + TILE) : a.S;  // shorter once the mask is read

  Stage<D> st;
  st.init(a.width, a.width);
  unsigned long long bits = 0, next = 0;
  int key = 0;
  auto fetch = [&](int c) {
    const unsigned to = (c & 1) * 2 * MAT;
    key = key_byte(mask, c * KC, end);
    st.load(k, a.width, v, a.width, c * KC, end, to, to + MAT);
  };
  auto arrive = [&](int c) {
    char* to = buf + (c & 1) * 2 * MAT;
    st.wait();
    next = __ballot(c * KC + lane < end && key != 0);
    st.clear(to, to + MAT, next);
  };
  // everything that the first chunk needs is on its way at once
  const int all = (end + KC - 1) / KC, first = __builtin_amdgcn_readfirstlane(all * span / a.q_spans);
  fetch(first);
  const Bias<> first_bias(a, h);
  if (mask) end = mask_end(mask, end, ends);
  const int chunks = min((end + KC - 1) / KC, all * (span + 1) / a.q_spans);
  // a row past the end, or with nothing allowed, takes part as zeros
  const float lse = i < a.S ? a.lse[(long long)bh * a.S + i] : INF;
  const float rest_p = a.lse[(long long)a.B * a.NH * a.S + (long long)bh * a.S + min(i, a.S - 1)];  // 1, or 1 / sum
  const bool live = lse < INF || lse != lse;
  b8 q[D / 16], g[D / 16];
  float dsum = 0.f;
  {
    const int r = min(i, a.S - 1);
    const __bf16* qp = a.qkv + ((long long)b * a.S + r) * a.width + h * D;
    const long long at = (((long long)b * a.S + r) * a.NH + h) * D;
    const b8 zero = {};
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      q[t] = *(const b8*)(qp + 16 * t + 8 * hi);
      g[t] = *(const b8*)(a.dout + at + 16 * t + 8 * hi);
      const b8 out = *(const b8*)(a.out + at + 16 * t + 8 * hi);
      q[t] = live ? q[t] : zero;
      g[t] = live ? g[t] : zero;
#pragma unroll
      for (int e = 0; e < 8; ++e) dsum = fmaf((float)g[t][e], (float)out[e], dsum);
    }
  }
  dsum += __shfl_xor(dsum, 32, 64);
  if (i < a.S && hi == 0 && span == 0) a.dsum[(long long)bh * a.S + i] = dsum;

  f16 dq[D / 32] = {};
  const float c2 = a.scale * LOG2E;
  float* mine = sums + (2 * wave + hi) * offs;
  float far_low = 0.f, far_high = 0.f;
  // This row's dS must sum to zero. It does not quite: D comes from out as it was
  // rounded, and what D is off by goes into a bucket with the bucket's share of P.
  // In one that holds most of P but sums to little (all keys beyond the largest
  // distance of a long sequence) that would be most of the result; so the row's
  // sum `rest` is taken out of the two outermost offsets by their share of P.
  float rest = 0.f, own_low = 0.f, own_high = 0.f, mass_low = 0.f, mass_high = 0.f;
  // The upper 32 offsets of a tile are the lower 32 of the next one: they wait in
  // a register. What is added to LDS goes to the half wave's own array, 32 lanes
  // to 32 offsets, so it needs no atomic (one costs as much as the tile's
  // products); offsets beyond the largest distance, where lanes would meet, stay
  // in registers.
  float left = 0.f;
  int left_at = i0;  // the key tile that `left` is for
  const int lane_off = 4 * hi - (lane & 31);
  auto add = [&](int d, float x) {
    far_low += d <= -a.far ? x : 0.f;
    far_high += d >= a.far ? x : 0.f;
    if (d > -a.far && d < a.far) mine[d + a.far] += x;
  };
  first_bias.put(a.scale, bias);
  for (int x = threadIdx.x; x < 8 * offs; x += 256) sums[x] = 0.f;
  st.wait();
  if (first < chunks) arrive(first);
  __syncthreads();
  const float low = shared(bias[0]), high = shared(bias[2 * a.far + 7]);
  const Flat flat_low(low, c2), flat_high(high, c2);
  dsum *= rest_p;

  for (int c = first; c < chunks; ++c) {
    bits = next;
    if (c > first) __syncthreads();
    if (c + 1 < chunks) fetch(c + 1);
    const char* kt = buf + (c & 1) * 2 * MAT;
    const char* vt = kt + MAT;
#pragma unroll 1  // one copy of the code: on short sequences its fetches are what is waited for
    for (int sub = 0; sub < 2; ++sub) {
      const int j0 = c * KC + 32 * sub;
      const unsigned on = (unsigned)(bits >> (32 * sub));
      if (on == 0 || (a.causal && j0 > i0 + 31)) continue;
      const char* ksub = kt + 64 * D * sub;
      const char* vsub = vt + 64 * D * sub;
      f16 s, dp = {};
      const bool beyond = j0 + 31 - i0 <= -a.far || j0 - (i0 + 31) >= a.far;
      float flat = 0.f, flat_lo = 0.f;  // as in the forward
      if (beyond) {
        flat = j0 < i0 ? flat_low.hi : flat_high.hi;
        flat_lo = j0 < i0 ? flat_low.lo : flat_high.lo;
        s = mfma(row_frag<D>(ksub, lane & 31, 0, hi), q[0], (f16){});
      } else {
        s = mfma(row_frag<D>(ksub, lane & 31, 0, hi), q[0], bias_tile(bias, a.far, j0, i0, lane, low, high));
      }
      dp = mfma(row_frag<D>(vsub, lane & 31, 0, hi), g[0], dp);
#pragma unroll
      for (int t = 1; t < D / 16; ++t) {
        s = mfma(row_frag<D>(ksub, lane & 31, t, hi), q[t], s);
        dp = mfma(row_frag<D>(vsub, lane & 31, t, hi), g[t], dp);
      }
      reads_ahead<D / 8 - 1>();
      const float base = flat - lse + flat_lo;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, base));
      drop_rows(s, on, a.causal && j0 + 31 > i0, j0, i0, lane, 0.f);
      float whole = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dp[r] = s[r] * fmaf(dp[r], rest_p, -dsum);
        whole += dp[r];
      }
      // sums of dS by offset: tiles beyond the largest distance in a register,
      // others along their diagonals
      rest += whole;
      if (beyond) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += s[r];
        const bool low_side = j0 < i0;
        own_low += low_side ? whole : 0.f;
        own_high += low_side ? 0.f : whole;
        mass_low += low_side ? t : 0.f;
        mass_high += low_side ? 0.f : t;
      } else {
        float d[3] = {};
        if (left_at != j0) add(left_at - i0 + lane_off, left);
        else d[0] = left;
        diagonals_32(dp, d, lane & 16);
        add(j0 - i0 + lane_off, d[0]);
        left = d[2];
        left_at = j0 + 32;
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const b8 p = pack(dp, ks);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dq[dt] = mfma(col_frag<D>(ksub, 16 * ks, dt, lane), p, dq[dt]);
      }
    }
    if (c + 1 < chunks) arrive(c + 1);
  }
  add(left_at - i0 + lane_off, left);
  rest += __shfl_xor(rest, 32, 64);
  mass_low *= rest_p;
  mass_high *= rest_p;
  if (a.q_spans > 1) {  // the row's sums are known to k_rel_dq
    const long long rows = (long long)a.B * a.NH * a.S, row = span * rows + (long long)bh * a.S + i;
    mass_low += __shfl_xor(mass_low, 32, 64);
    mass_high += __shfl_xor(mass_high, 32, 64);
    if (i < a.S) {
      store_columns<D>(a.dq + row * D, dq, a.scale, hi);
      if (hi == 0) *(f4*)(a.dq + a.q_spans * rows * D + row * 4) = f4{rest, mass_low, mass_high, 0.f};
    }
    rest = 0.f;
  }
  far_low += fmaf(-rest, mass_low, own_low);  // each half takes its own share
  far_high += fmaf(-rest, mass_high, own_high);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) {
    far_low += __shfl_xor(far_low, x, 64);
    far_high += __shfl_xor(far_high, x, 64);
  }
  if (lane == 0) {
    mine[0] += far_low;
    mine[offs - 1] += far_high;
  }
  __syncthreads();
  if (a.q_spans == 1)
    store_rows<D>(smem + wave * 64 * D, a.dqkv + ((long long)b * a.S + i0) * a.width + h * D, a.width, a.S - i0, dq, a.scale, lane);
  float* to = a.doff + (((long long)h * a.B + b) * rel_doff_rows(a.S, a.q_spans) + tile * a.q_spans + span) * offs;
  for (int x = threadIdx.x; x < offs; x += 256) {
    float t = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) t += sums[n * offs + x];
    to[x] = t;
  }
}

// Joins the spans: dQ, four columns a thread, in order; and in the first workgroups,
// one for 128 rows, what the rows' sums take out of the two outermost offsets, as
// one more row of offsets' sums (5.5 us).
template <int D>
__global__ __launch_bounds__(256) void k_rel_dq(RelArgs a, int tiles) {
  __shared__ float lds[2][2];
  const long long rows = (long long)a.B * a.NH * a.S;
  const int sums = a.B * a.NH * tiles;
  if ((int)blockIdx.x >= sums) {
    const long long row = (long long)(blockIdx.x - sums) * (1024 / D) + threadIdx.x / (D / 4);
    const int d = threadIdx.x % (D / 4) * 4;
    if (row >= rows) return;
    f4 t = {};
    for (int s = 0; s < a.q_spans; ++s) t += *(const f4*)(a.dq + (s * rows + row) * D + d);
    b4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (__bf16)t[e];
    const int i = (int)(row % a.S), h = (int)(row / a.S % a.NH);
    const long long b = row / a.S / a.NH;
    *(b4*)(a.dqkv + (b * a.S + i) * a.width + h * D + d) = v;
    return;
  }
  const int tile = blockIdx.x % tiles, bh = blockIdx.x / tiles, h = bh % a.NH, b = bh / a.NH;
  const int i = tile * TILE + threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float low = 0.f, high = 0.f;
  if (threadIdx.x < TILE && i < a.S) {
    f4 t = {};
    for (int s = 0; s < a.q_spans; ++s) t += *(const f4*)(a.dq + a.q_spans * rows * D + (s * rows + (long long)bh * a.S + i) * 4);
    low = -t[0] * t[1];
    high = -t[0] * t[2];
  }
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) {
    low += __shfl_xor(low, x, 64);
    high += __shfl_xor(high, x, 64);
  }
  if (lane == 0 && wave < 2) {
    lds[wave][0] = low;
    lds[wave][1] = high;
  }
  __syncthreads();
  const int offs = 2 * a.far + 1;
  float* to = a.doff + (((long long)h * a.B + b) * rel_doff_rows(a.S, a.q_spans) + tiles * a.q_spans + tile) * offs;
  for (int x = threadIdx.x; x < offs; x += 256)
    to[x] = x == 0 ? lds[0][0] + lds[1][0] : x == offs - 1 ? lds[0][1] + lds[1][1] : 0.f;
}

// dtable[n][h]: the offsets' sums over batches and tiles, then over the offsets
// of a bucket; one workgroup a head, every sum in a fixed order. It needs the
// dQ kernel alone, so it runs beside dK and dV, as their kernel's first NH
// workgroups (as a kernel of its own behind them it took 4 to 14 us).
template <int T>
__device__ void sum_table(const RelArgs& a, int h, char* smem) {
  constexpr int W = T / 64, COLS = 320;
  float* part = (float*)smem;                                // [W][COLS]
  float* sums = part + W * COLS;                             // [2 * far + 1]
  short* map = (short*)(sums + 2 * GA_REL_MAX_DISTANCE + 1);  // [2 * far + 1]
  const int offs = 2 * a.far + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = a.B * rel_doff_rows(a.S, a.q_spans);
  const float* p = a.doff + (long long)h * n * offs;
  for (int x = threadIdx.x; x < offs; x += T) map[x] = (short)min(max(a.map[x], 0), a.buckets - 1);
  for (int x0 = 0; x0 < offs; x0 += COLS) {
    float t[5] = {};
#pragma unroll 4
    for (int w = wave; w < n; w += W) {
#pragma unroll
      for (int i = 0; i < 5; ++i) t[i] += p[(long long)w * offs + min(x0 + 64 * i + lane, offs - 1)];
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) part[wave * COLS + 64 * i + lane] = t[i];
    __syncthreads();
    for (int x = threadIdx.x; x < COLS && x0 + x < offs; x += T) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) s += part[i * COLS + x];
      sums[x0 + x] = s;
    }
    __syncthreads();
  }
  for (int bucket = wave; bucket < a.buckets; bucket += W) {
    float t = 0.f;
    for (int e = lane; e < offs; e += 64)
      if (map[e] == bucket) t += sums[e];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    if (lane == 0) a.dtable[(long long)bucket * a.NH + h] = (__bf16)t;
  }
}

// ---------------- backward 2: dK and dV; a wave owns 32 keys, chunks of 64 queries ----------------
// Registers decide here: dK, dV, K and V of 32 keys are 256 of them at head size
// 128. V is kept in LDS there, by eight waves that share a chunk instead of four:
// two waves a SIMD (long: 480 us with V in registers, 340 so, when that step was
// taken; padded: 45 us with V in registers, 61 in LDS with four waves, 85 with
// eight). padded 42 us (matrix unit 22 % busy), long 294 us (43 %, 934 TFLOP/s),
// the table's sums among them.
template <int D>
constexpr int kv_waves() { return D == 64 ? 4 : 8; }
template <int D>
__global__ __launch_bounds__(64 * kv_waves<D>(), D == 64 ? 3 : 2) void k_rel_bwd_kv(RelArgs a, int tiles) {
  constexpr int T = 64 * kv_waves<D>(), KEYS = T / 2;
  constexpr bool V_LDS = D == 128;
  extern __shared__ __align__(16) char smem[];  // the chunks lie in the first 64 KB, which m0 reaches
  char* buf = smem;                             // [2][Q, dO]
  constexpr int MAT = KC * 2 * D;
  float* rows = (float*)(smem + 4 * MAT);    // [2][lse, -D][64]
  char* vt = (char*)(rows + 4 * KC);         // V_LDS: [KEYS][D]
  float* bias = (float*)(vt + (V_LDS ? KEYS * 2 * D : 0));

  if ((int)blockIdx.x < a.NH) return sum_table<T>(a, blockIdx.x, smem);
  int tile;
  const int column = place(blockIdx.x - a.NH, a.B * a.NKV, a.parts, tiles, a.causal || a.mask, tile);  // the first tile has the most queries, and keys that count
  const int part = column % a.parts, bk = column / a.parts;
  const int heads = a.parts / a.spans, part_h = part % heads, span = part / heads;  // every heads-th query head, a span of the queries
  const int hk = bk % a.NKV, b = bk / a.NKV, group = a.NH / a.NKV;
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int row = (threadIdx.x >> 6) * 32 + (lane & 31);  // of the tile's keys
  const int j0 = tile * KEYS + (threadIdx.x >> 6) * 32, j = j0 + (lane & 31);
  const bool keep = j < a.S && (!a.mask || a.mask[(long long)b * a.S + min(j, a.S - 1)]);
  const bool work = __any(keep);  // this wave has a key that counts

  const int from = a.causal ? tile * KEYS / KC : 0, chunks = (a.S + KC - 1) / KC - from;
  const int first = from + chunks * span / a.spans, end = from + chunks * (span + 1) / a.spans;
  Stage<D, T> st;
  st.init(a.width, a.NH * D);
  float row_lse = 0.f, row_d = 0.f;
  const __bf16 *q, *g;
  const float *lse, *dsum;
  auto fetch = [&](int c) {
    const unsigned to = (c & 1) * 2 * MAT;
    const int r = c * KC + lane;
    row_lse = lse[min(r, a.S - 1)];
    row_d = dsum[min(r, a.S - 1)];
    st.load(q, a.width, g, a.NH * D, c * KC, a.S, to, to + MAT);
  };
  auto put = [&](int c) {
    char* to = buf + (c & 1) * 2 * MAT;
    st.wait();
    if (c * KC + lane >= a.S) row_lse = INF, row_d = 0.f;
    st.clear(to, to + MAT, __ballot(row_lse < INF || row_lse != row_lse));  // rows with nothing allowed too
    if (__any(fabsf(row_lse) >= LARGE && row_lse < INF)) {
      // the factor of P that stands apart goes into dO and D, rounding dO once more: dV takes P dO, dK takes P (dP - D)
      const float* rest = lse + (long long)a.B * a.NH * a.S;
      row_d *= rest[min(c * KC + lane, a.S - 1)];
      st.scale(to + MAT, rest, c * KC, a.S);
    }
    if (threadIdx.x < KC) {
      float* r = rows + (c & 1) * 2 * KC;
      r[threadIdx.x] = row_lse;
      r[KC + threadIdx.x] = -row_d;
    }
  };
  auto begin = [&](int n) {  // the first chunk and the bias of the n-th query head are on their way
    const int h = hk * group + n;
    q = a.qkv + (long long)b * a.S * a.width + h * D;
    g = a.dout + ((long long)b * a.S * a.NH + h) * D;
    lse = a.lse + (long long)(b * a.NH + h) * a.S;
    dsum = a.dsum + (long long)(b * a.NH + h) * a.S;
    fetch(first);
    return Bias<T, true>(a, h);
  };
  auto next = begin(part_h);

  b8 k[D / 16], v[V_LDS ? 1 : D / 16];
  {
    const int r = min(j, a.S - 1);
    const __bf16* kp = a.qkv + ((long long)b * a.S + r) * a.width + (a.NH + hk) * D;
    const __bf16* vp = kp + a.NKV * D;
    const b8 zero = {};
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      k[t] = *(const b8*)(kp + 16 * t + 8 * hi);
      const b8 x = *(const b8*)(vp + 16 * t + 8 * hi);
      k[t] = keep ? k[t] : zero;
      if (V_LDS) *(b8*)(vt + piece<D>(row, 2 * t + hi)) = keep ? x : zero;  // read by this wave alone
      else v[V_LDS ? 0 : t] = keep ? x : zero;
    }
  }
  f16 dk[D / 32] = {}, dv[D / 32] = {};
  const float c2 = a.scale * LOG2E;
  st.wait();

  if (__syncthreads_or(work))
    for (int n = part_h; n < group; n += heads) {
      if (n != part_h) {
        __syncthreads();  // the last head's tiles are read
        next = begin(n);
      }
      next.put(a.scale, bias);
      put(first);
      __syncthreads();
      const float low = shared(bias[0]), high = shared(bias[2 * a.far + 7]);
      for (int c = first; c < end; ++c) {
        if (c > first) __syncthreads();
        if (c + 1 < end) fetch(c + 1);
        const char* qt = buf + (c & 1) * 2 * MAT;
        const char* gt = qt + MAT;
        const float* rl = rows + (c & 1) * 2 * KC;
#pragma unroll 1
        for (int sub = 0; sub < 2; ++sub) {
          const int i0 = c * KC + 32 * sub;
          if (!work || i0 >= a.S || (a.causal && i0 + 31 < j0)) continue;
          const char* qs = qt + 64 * D * sub;
          const char* gs = gt + 64 * D * sub;
          // rows are queries here: the mirrored bias of row - column
          f16 s = bias_tile(bias, a.far, i0, j0, lane, low, high), dp;  // dP starts from -D: no subtraction later
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const f4 d = *(const f4*)(rl + KC + 32 * sub + 8 * x + 4 * hi);
#pragma unroll
            for (int y = 0; y < 4; ++y) dp[4 * x + y] = d[y];
          }
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            s = mfma(row_frag<D>(qs, lane & 31, t, hi), k[t], s);
            dp = mfma(row_frag<D>(gs, lane & 31, t, hi), V_LDS ? row_frag<D>(vt, row, t, hi) : v[V_LDS ? 0 : t], dp);
          }
          if (!V_LDS) reads_ahead<D / 8>();
          if (a.causal && i0 < j0 + 31) {
            asm volatile("");
            const int least = j - i0 - 4 * hi;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = crow(r, 0) >= least ? s[r] : -INF;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const f4 e = *(const f4*)(rl + 32 * sub + 8 * x + 4 * hi);
#pragma unroll
            for (int y = 0; y < 4; ++y) s[4 * x + y] = __builtin_amdgcn_exp2f(fmaf(s[4 * x + y], c2, -e[y]));
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= s[r];
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const b8 p = pack(s, ks), ds = pack(dp, ks);
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) {
              dv[dt] = mfma(col_frag<D>(gs, 16 * ks, dt, lane), p, dv[dt]);
              dk[dt] = mfma(col_frag<D>(qs, 16 * ks, dt, lane), ds, dk[dt]);
            }
          }
        }
        if (c + 1 < end) put(c + 1);
      }
    }
  // a masked key's column holds what its zeroed K and V gave: it has no gradient
  if (!keep)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) dk[dt] = dv[dt] = (f16){};
  if (a.parts > 1) {
    if (j >= a.S) return;
    float* to = a.dkv + (((long long)part * a.B * a.NKV + bk) * a.S + j) * 2 * D;
    store_columns<D>(to, dk, a.scale, hi);
    store_columns<D>(to + D, dv, 1.f, hi);
  } else {
    __syncthreads();  // the chunks are read
    char* own = smem + (threadIdx.x >> 6) * 64 * D;
    __bf16* to = a.dqkv + ((long long)b * a.S + j0) * a.width + (a.NH + hk) * D;
    store_rows<D>(own, to, a.width, a.S - j0, dk, a.scale, lane);
    store_rows<D>(own, to + a.NKV * D, a.width, a.S - j0, dv, 1.f, lane);
  }
}

// the parts' dK and dV, added in order: four columns a thread; long 24 us (151 MB)
__global__ __launch_bounds__(256) void k_rel_dkv(RelArgs a, long long n) {
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= n) return;
  const int per = a.D / 2, c = (int)(x % per) * 4;  // of [dK, dV], 2 D columns
  const long long row = x / per, part = (long long)a.B * a.NKV * a.S * 2 * a.D;
  const float* p = a.dkv + row * 2 * a.D + c;
  f4 t = *(const f4*)p;
  for (int i = 1; i < a.parts; ++i) t += *(const f4*)(p + i * part);
  b4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (__bf16)t[e];
  const int s = (int)(row % a.S), hk = (int)(row / a.S % a.NKV);
  const long long b = row / a.S / a.NKV;
  const int head = c < a.D ? a.NH + hk : a.NH + a.NKV + hk;
  *(b4*)(a.dqkv + (b * a.S + s) * a.width + head * a.D + c % a.D) = v;
}

// ---------------- new tokens over a cache ----------------
// The columns of a wave's tile are the rows (new token, head of the group) that
// share a key/value head: one read of K and V serves them all. The keys are
// split over `splits` workgroups and eight waves each (with four, 4x512 took 9.0 us
// instead of 7.5); a wave takes 32 keys at a time, K straight into A fragments, V
// through its own LDS tile. The waves' (maximum, sum, output) are joined in LDS,
// the workgroups' by k_rel_join. Bound by the cache's bytes: 16 sequences of up to
// 16384 tokens, 16 heads over 4, D 128: 88 to 91 us with the join, 4.4 to 4.6 TB/s
// of the 4.9 that a copy reaches.
constexpr int TOKEN_WAVES = 8;
template <int D>
__global__ __launch_bounds__(512) void k_rel_token(RelTokenArgs a, int row_tiles) {
  constexpr int W = TOKEN_WAVES, T = 64 * W;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int group = a.NH / a.NKV, rows = group * a.Sq;
  const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int rt = rest % row_tiles, hk = rest / row_tiles % a.NKV, b = rest / row_tiles / a.NKV;
  constexpr int MAT = 32 * 2 * D;
  char* vt = smem + wave * MAT;
  int* map = (int*)(smem + W * MAT);             // [far + 1], offsets -far .. 0
  float* table = (float*)(map + a.far + 1);      // [buckets][heads of this tile]
  const int row = rt * 32 + (lane & 31);
  const int tok = min(row, rows - 1) / group, h = hk * group + min(row, rows - 1) % group;
  const int len = min(max(a.lengths[b], 0), a.S);
  const int pos = row < rows ? len - a.Sq + tok : -1;  // the last key of this row
  const int pos0 = len - a.Sq + rt * 32 / group;       // the first row's

  // keys in units of 32, spread evenly over the waves of all splits
  const int units = (len + 31) / 32, waves = a.splits * W, w = split * W + wave;
  const int u0 = (int)((long long)units * w / waves), u1 = (int)((long long)units * (w + 1) / waves);
  const __bf16* k = a.k + b * a.k_b + hk * a.k_h;
  const __bf16* v = a.v + b * a.v_b + hk * a.v_h;
  constexpr int NV = 32 * D / 8 / 64;
  b8 kf[D / 16], vf[NV];
  auto fetch = [&](int u) {
    const int j = u * 32 + (lane & 31);
    const __bf16* kp = k + min(j, len - 1) * a.k_s;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) kf[t] = *(const b8*)(kp + 16 * t + 8 * hi);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int x = lane + 64 * n, r = u * 32 + x / (D / 8);
      vf[n] = *(const b8*)(v + min(r, len - 1) * a.v_s + x % (D / 8) * 8);
    }
  };
  // the first keys are on their way while the bias is staged
  if (u0 < u1) fetch(u0);
  b8 q[D / 16];
  const __bf16* qp = a.q + b * a.q_b + tok * a.q_s + h * a.q_h;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) q[t] = *(const b8*)(qp + 16 * t + 8 * hi);
  for (int x = threadIdx.x; x <= a.far; x += T) map[x] = min(max(a.map[x], 0), a.buckets - 1);
  for (int x = threadIdx.x; x < a.buckets * group; x += T)
    table[x] = as_bias(a.table[(long long)(x / group) * a.NH + hk * group + x % group], a.scale);
  __syncthreads();
  const int mine = h - hk * group;
  const float low = table[map[0] * group + mine];

  f16 o[D / 32] = {};
  float m = -INF, l = 0.f;
  const float c2 = a.scale * LOG2E;
  for (int u = u0; u < u1; ++u) {
    const int j0 = u * 32;
    const b8 zero = {};
    f16 s;
    if (j0 + 31 - pos0 <= -a.far) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = low;
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = j0 + crow(r, hi) - pos;
        s[r] = table[map[min(max(d, -a.far), 0) + a.far] * group + mine];
      }
    }
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      const b8 f = j0 + (lane & 31) < len ? kf[t] : zero;
      s = mfma(f, q[t], s);
    }
    // this tile's V into LDS; the wave alone reads it
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int x = lane + 64 * n, r = x / (D / 8);
      *(b8*)(vt + piece<D>(r, x % (D / 8))) = j0 + r < len ? vf[n] : zero;
    }
    if (u + 1 < u1) fetch(u + 1);
    if (j0 + 31 > pos0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = j0 + crow(r, hi) <= pos ? s[r] : -INF;
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64)) * c2;
    if (__any(top > m + 8.f)) {
      const float n = fmaxf(m, top);
      const float f = n == -INF ? 1.f : __builtin_amdgcn_exp2f(m - n);
      m = n;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= f;
    }
    const float base = m == -INF ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, -base));
      l += s[r];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const b8 p = pack(s, ks);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] = mfma(col_frag<D>(vt, 16 * ks, dt, lane), p, o[dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  l += __shfl_xor(l, 32, 64);

  // join the waves, eight rows at a time: [W][maximum, sum][32], the rows' own, [W][8][D + 4]
  __syncthreads();
  float* stat = (float*)smem;
  float* stats = stat + W * 64;
  float* acc = stats + 64;
  if (hi == 0) {
    stat[wave * 64 + lane] = m;
    stat[wave * 64 + 32 + lane] = l;
  }
  __syncthreads();
  const int x = lane & 31;
  float top = -INF, sum = 0.f;
#pragma unroll
  for (int n = 0; n < W; ++n) top = fmaxf(top, stat[n * 64 + x]);
  const float base = top == -INF ? 0.f : top;
#pragma unroll
  for (int n = 0; n < W; ++n) sum += stat[n * 64 + 32 + x] * __builtin_amdgcn_exp2f(stat[n * 64 + x] - base);
  const float f = __builtin_amdgcn_exp2f(m - base);
  if (threadIdx.x < 32) {
    stats[threadIdx.x] = top;
    stats[32 + threadIdx.x] = sum;
  }
  const int count = min(rows - rt * 32, 32);
  for (int r0 = 0; r0 < count; r0 += 8) {
    if (r0 > 0) __syncthreads();
    if (x >= r0 && x < min(r0 + 8, count)) store_columns<D>(acc + (wave * 8 + x - r0) * (D + 4), o, f, hi);
    __syncthreads();
    for (int e = threadIdx.x; e < 8 * D; e += T) {
      const int r = r0 + e / D, d = e % D, at = rt * 32 + r;
      if (r >= count) break;
      float t = 0.f;
#pragma unroll
      for (int n = 0; n < W; ++n) t += acc[(n * 8 + r - r0) * (D + 4) + d];
      if (a.splits == 1) {
        const float z = stats[32 + r];
        a.out[(((long long)b * a.Sq + at / group) * a.NH + hk * group + at % group) * D + d] = (__bf16)(z == 0.f ? 0.f : t / z);
      } else {
        float* p = a.parts + (((long long)rest * a.splits + split) * 32 + r) * (D + 2);
        p[d] = t;
        if (d == 0) {
          p[D] = stats[r];
          p[D + 1] = stats[32 + r];
        }
      }
    }
  }
}

// joins the workgroups' parts of one output row, in order (4.9 us at 256 rows of 8 parts, D 128)
template <int D>
__global__ __launch_bounds__(D) void k_rel_join(RelTokenArgs a, int row_tiles) {
  const int group = a.NH / a.NKV, rows = group * a.Sq;
  const int at = blockIdx.x % rows, hk = blockIdx.x / rows % a.NKV, b = blockIdx.x / rows / a.NKV;
  const long long rest = ((long long)b * a.NKV + hk) * row_tiles + at / 32;
  const float* p = a.parts + (rest * a.splits * 32 + at % 32) * (D + 2);
  const long long step = 32 * (D + 2);
  // every thread holds its column of up to 16 parts at a time, so that their
  // loads are in flight together
  float top = -INF, z = 0.f, o = 0.f;
  for (int n0 = 0; n0 < a.splits; n0 += 16) {
    float m[16], l[16], x[16], more = top;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const float* at_n = p + min(n0 + n, a.splits - 1) * step;
      m[n] = n0 + n < a.splits ? at_n[D] : -INF;
      l[n] = at_n[D + 1];
      x[n] = at_n[threadIdx.x];
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) more = larger(more, m[n]);
    const float base = more == -INF ? 0.f : more, f = __builtin_amdgcn_exp2f(top - base);
    z *= f;
    o *= f;
    top = more;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const float g = __builtin_amdgcn_exp2f(m[n] - base);
      z = fmaf(l[n], g, z);
      o = fmaf(x[n], g, o);
    }
  }
  a.out[(((long long)b * a.Sq + at / group) * a.NH + hk * group + at % group) * D + threadIdx.x] =
      (__bf16)(z == 0.f ? 0.f : o / z);
}

size_t bias_bytes(int far) { return 16 * (size_t)bias_len(far); }

// dynamic LDS above 64 KB has to be asked for
template <typename F>
hipError_t allow(F* f, size_t bytes) {
  if (bytes <= 64 * 1024) return hipSuccess;
  return hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <int D>
hipError_t forward(const RelArgs& a, hipStream_t s) {
  const int tiles = rel_tiles(a.S);
  const size_t lds = 4 * KC * 2 * D + bias_bytes(a.far) + 16;
  hipError_t e = allow(k_rel_fwd<D>, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_rel_fwd<D>), dim3(a.B * a.NH * tiles * a.spans), dim3(256), lds, s, a, tiles);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (a.spans > 1) {
    const long long rows = (long long)a.B * a.NH * a.S;
    hipLaunchKernelGGL((k_rel_out<D>), dim3((unsigned)((rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <int D>
hipError_t backward(const RelArgs& a, hipStream_t s) {
  const int tiles = rel_tiles(a.S);
  const size_t lds_q = 4 * KC * 2 * D + bias_bytes(a.far) + 16 + 32 * (2 * a.far + 1);
  constexpr int T = 64 * kv_waves<D>();
  const int kv_tiles = (a.S + T / 2 - 1) / (T / 2);
  const size_t lds_kv = 4 * KC * 2 * D + 16 * KC + (D == 128 ? T * D : 0) + bias_bytes(a.far);
  hipError_t e = allow(k_rel_bwd_q<D>, lds_q);
  if (e == hipSuccess) e = allow(k_rel_bwd_kv<D>, lds_kv);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_rel_bwd_q<D>), dim3(a.B * a.NH * tiles * a.q_spans), dim3(256), lds_q, s, a, tiles);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (a.q_spans > 1) {
    const long long rows = (long long)a.B * a.NH * a.S;
    hipLaunchKernelGGL((k_rel_dq<D>), dim3((unsigned)(a.B * a.NH * tiles + (rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, s, a, tiles);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_rel_bwd_kv<D>), dim3(a.NH + a.B * a.NKV * a.parts * kv_tiles), dim3(T), lds_kv, s, a, kv_tiles);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (a.parts > 1) {
    const long long n = (long long)a.B * a.NKV * a.S * (D / 2);
    hipLaunchKernelGGL(k_rel_dkv, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a, n);
  }
  return hipGetLastError();
}

template <int D>
hipError_t token(const RelTokenArgs& a, hipStream_t s) {
  constexpr int W = TOKEN_WAVES;
  const int group = a.NH / a.NKV, rows = group * a.Sq, row_tiles = (rows + 31) / 32;
  static_assert(4 * (W * 64 + 64 + W * 8 * (D + 4)) <= W * 32 * 2 * D, "the join fits where V was");
  const size_t lds = W * 32 * 2 * D + 4 * (a.far + 1) + 4 * (size_t)a.buckets * group;
  const hipError_t e = allow(k_rel_token<D>, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_rel_token<D>), dim3(a.B * a.NKV * row_tiles * a.splits), dim3(64 * W), lds, s, a, row_tiles);
  if (a.splits > 1) hipLaunchKernelGGL((k_rel_join<D>), dim3(a.B * a.NKV * rows), dim3(D), 0, s, a, row_tiles);
  return hipGetLastError();
}

}  // namespace

// Over how many workgroups the keys of a tile of queries are cut where there are
// few tiles, of at least five chunks each. With their joining kernels, forward and
// dQ: 1x4000, 2 heads, D 128 88 -> 38 and 147 -> 57 us; 2x1042 causal, 4 heads, D 128
// 28 -> 22 and 44 -> 32; 1x2000, 8 heads, D 64 37 -> 28 and 62 -> 46. In two spans of
// four chunks 1x512 would lose (13 -> 14 and 22 -> 23).
int rel_spans(int B, int S, int NH) {
  const long long base = (long long)B * NH * rel_tiles(S);
  int n = 1;
  while (base * (n + 1) <= 256 && (S + KC - 1) / KC >= 5 * (n + 1)) ++n;
  return n;
}

// Over how many workgroups the query heads that share a key/value head are
// spread in the backward: one workgroup walks all queries of its heads, so
// with few of them (and uneven ones, under the causal mask) the chip waits for
// the longest. Where that leaves compute units without one, the queries are cut
// into spans too, of at least four chunks: 1x4000, 2 heads, D 128 222 -> 57 us and
// 12 for k_rel_dkv, 2x1042 causal, 4 heads, D 128 66 -> 38 and 9, 1x512, 8 heads,
// D 64 23 -> 18 and 4.
void rel_parts(int B, int S, int NH, int NKV, int D, int* parts, int* spans) {
  const int group = NH / NKV, tiles = rel_tiles(S);
  int n = 1;
  while (n < group && (long long)B * NKV * tiles * n < 1024) ++n;
  while (group % n) ++n;
  const int keys = D == 64 ? 32 * kv_waves<64>() : 32 * kv_waves<128>();
  const long long base = (long long)B * NKV * n * ((S + keys - 1) / keys);
  int m = 1;
  while (base * (m + 1) <= 256 && (S + KC - 1) / KC >= 4 * (m + 1)) ++m;
  *parts = n * m;
  *spans = m;
}

// Enough workgroups to fill the chip, but at least 64 keys a wave, since a second
// kernel joins the parts: with 32, 4x512 (8 heads, D 64) takes 8.7 us instead of
// 7.5, 4x1000 (8 heads over 2) 8.7 instead of 9.8; with 128, 1x16000 (8 over 1)
// 12.4 instead of 10.9. Sequences differ in length, so workgroups of 4096 keys and
// more are cut further: 16 sequences of 1 to 16384 tokens, 16 heads over 4, D 128:
// 62 -> 54 us (8 over 8, D 64: 65 -> 52); 16x4096 would lose by it (18 -> 20).
int rel_token_splits(int B, int Sq, int S, int NH, int NKV) {
  const long long rows = (long long)(NH / NKV) * Sq, base = (long long)B * NKV * ((rows + 31) / 32);
  long long n = (256 + base - 1) / base;
  const long long most = (S + 511) / 512;
  if (n > most) n = most;
  while (n * 4096 <= S && base * n < 1024) n *= 2;
  return (int)(n < 1 ? 1 : n);
}

hipError_t rel_forward(const RelArgs& a, hipStream_t s) { return a.D == 64 ? forward<64>(a, s) : forward<128>(a, s); }
hipError_t rel_backward(const RelArgs& a, hipStream_t s) { return a.D == 64 ? backward<64>(a, s) : backward<128>(a, s); }
hipError_t rel_token(const RelTokenArgs& a, hipStream_t s) { return a.D == 64 ? token<64>(a, s) : token<128>(a, s); }
