// "pages_write_*": rows of keys and values into the pages of a batch, quantized; "pages_read_*": rows of pages as fp32 or fp16.

#include <type_traits>

#include "pages.hpp"
#include "qmm_kernels.hpp"

namespace qmm {
namespace {

// ---- codes ---------------------------------------------------------------------------------------
//
// x / scale to the nearest code, ties to the even one; code times scale.  Both are fp32 operations rounded once, so that a row
// written and read is a matter of definition, not of order.
template <PageKind KIND>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float scale) {
  constexpr float M = page_largest(KIND);
  auto of = [&](float v) { return fminf(fmaxf(v / scale, -M), M); };
  if constexpr (KIND == PageKind::Q8) {
    auto code = [&](float v) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(of(v)))) & 255u; };
    return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
  } else {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(of(a), of(b), 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(of(c), of(d), low, true));
  }
}
template <PageKind KIND>
__device__ __forceinline__ float decode(uint32_t four, int i) {
  if constexpr (KIND == PageKind::Q8) return static_cast<float>(static_cast<int>(four << (24 - 8 * i)) >> 24);
  switch (i) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(four), 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(four), 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(four), 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(four), 3);
  }
}

// ---- a page of the batch -------------------------------------------------------------------------
//
// A workgroup takes the keys or the values of a page and key head.  A page is written as a whole by one workgroup, so that its scale
// needs no second launch: new rows lie at places `from` .. `to` - 1 of it, places below `from` hold earlier positions.
struct PageWork {
  PageUnit unit;
  uint32_t kv, page, from, to, first_row;   // first_row: the call's row at place `from`
  bool values;
};
__device__ __forceinline__ bool page_work(const PageBatch& b, PageWork* w) {
  const uint32_t which = blockIdx.x % (2u * b.kv_heads);
  if (!find_unit(b, blockIdx.x / (2u * b.kv_heads), [&](const PageSequence& q) { return touched_pages(b, q); }, &w->unit)) return false;
  const PageSequence& q = w->unit.seq;
  const uint32_t block = 1u << b.log_block, past = q.len - q.rows, slot = (past >> b.log_block) + w->unit.at, base = slot << b.log_block;
  w->values = which >= b.kv_heads, w->kv = w->values ? which - b.kv_heads : which;
  w->from = past > base ? past - base : 0u;
  w->to = q.len - base < block ? q.len - base : block;
  w->first_row = q.first + (base + w->from - past);
  // (a vector load, so that what comes before its use is not kept waiting as by a scalar one)
  uint32_t here = 0u;
  asm("" : "+v"(here));
  w->page = b.table[static_cast<uint64_t>(w->unit.s) * b.width + slot + here];
  return true;
}

// Thread t's runs of sixteen bytes of a page: keys by (place, sixteen elements), values by (sixteen places, element), an element a
// lane, so that a wavefront's loads of rows are whole lines.
constexpr uint32_t kPageThreads = 256;

// Bound by memory: 8 bytes a row's element in, 2 out, and what a page that is continued holds.  A thread holds its ITEMS runs' rows from
// the search for the largest on, so that they are read once.  3300 rows of 8 heads of 128 in three sequences: 9 us (read twice: 12), 34 MB; one
// row: 4.5, three ways to memory one after the other.
template <PageKind KIND, int ITEMS>
__global__ __launch_bounds__(kPageThreads) void pages_write_kernel(PageBatch b, const float* __restrict__ k, const float* __restrict__ v, uint64_t k_stride,
                                                                   uint64_t v_stride, uint8_t* kp, uint8_t* vp, float* ks, float* vs) {
  __shared__ uint32_t most_of[kPageThreads / 64];
  PageWork w;
  if (!page_work(b, &w)) return;                          // workgroup-uniform
  const uint32_t t = threadIdx.x, D = b.head_dim, block = 1u << b.log_block, runs = D / 16u;
  const uint64_t stride = w.values ? v_stride : k_stride;
  const float* rows = (w.values ? v : k) + static_cast<uint64_t>(w.first_row) * stride + w.kv * D;   // of place `from`

  // A thread's n-th run: of a key's elements d .. d + 15 at `place`, or of an element d at places place .. place + 15.
  const uint32_t count = block * runs, of_row = (1u << 20) / (w.values ? D : runs) + 1u;      // (i < 2048 is divided by its product)
  struct Run {
    uint32_t i, place, d;
  };
  auto run_of = [&](int n) {
    const uint32_t i = t + static_cast<uint32_t>(n) * kPageThreads, row = i * of_row >> 20;
    return w.values ? Run{i, row * 16u, i - row * D} : Run{i, row, (i - row * runs) * 16u};
  };
  const uint32_t rows_here = w.to - w.from;
  float x[ITEMS][16];
  uint32_t most = 0u;                                      // the largest magnitude by its bits: infinities and NaN are above all numbers
#pragma unroll
  for (int n = 0; n < ITEMS; ++n) {
    const Run r = run_of(n);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[n][e] = 0.0f;
    if (!w.values) {
      if (r.i < count && r.place - w.from < rows_here) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 four = *reinterpret_cast<const float4*>(rows + (r.place - w.from) * stride + r.d + e);
          x[n][e] = four.x, x[n][e + 1] = four.y, x[n][e + 2] = four.z, x[n][e + 3] = four.w;
        }
      }
    } else if (r.i < count && r.place + 15u >= w.from && r.place < w.to) {
      // (places that hold no new row: another one's, so that no load has a condition, and then nothing)
#pragma unroll
      for (uint32_t e = 0; e < 16u; ++e) {
        const uint32_t at = r.place + e - w.from;          // (before the first: far above the last)
        x[n][e] = rows[(at < rows_here ? at : 0u) * stride + r.d];
      }
#pragma unroll
      for (uint32_t e = 0; e < 16u; ++e) x[n][e] = r.place + e - w.from < rows_here ? x[n][e] : 0.0f;
    }
  }
  // (the page's number is asked for before the rows and looked at behind them)
  const uint32_t page = __builtin_amdgcn_readfirstlane(w.page);
  if (page >= b.pages) return;                             // workgroup-uniform
  const uint64_t head = static_cast<uint64_t>(page) * b.kv_heads + w.kv;
  float* scale_at = (w.values ? vs : ks) + head;
  uint8_t* codes = (w.values ? vp : kp) + head * (static_cast<uint64_t>(block) * D);
  const float before = w.from == 0u ? 0.0f : *scale_at;
#pragma unroll
  for (int n = 0; n < ITEMS; ++n) {
#pragma unroll
    for (int e = 0; e < 16; ++e) most = max(most, bit_cast<uint32_t>(x[n][e]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (uint32_t off = 32u; off > 0u; off >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(most, off, kWave)));
  if ((t & 63u) == 0u) most_of[t >> 6] = most;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kPageThreads / 64u; ++i) most = max(most, most_of[i]);
  const float own = bit_cast<float>(most) / page_largest(KIND);
  // A page with an infinity or NaN is NaN until it is begun anew.
  const bool finite = most < 0x7F800000u && before < INFINITY && before >= 0.0f;
  const float scale = finite ? fmaxf(before, own) : bit_cast<float>(0x7FC00000u);
  if (t == 0u) *scale_at = scale;
  const bool empty = !(scale > 0.0f);                      // (NaN too): all codes 0
  const bool again = w.from != 0u && (empty || scale != before);      // codes that were there change
#pragma unroll
  for (int n = 0; n < ITEMS; ++n) {
    const Run r = run_of(n);
    const uint32_t old_places = r.place >= w.from ? 0u : w.values ? w.from - r.place : 1u;      // of the run's, that held codes (16 and more: all)
    if (r.i >= count || (!again && (w.values ? old_places >= 16u : old_places != 0u))) continue;
    uint4* to = reinterpret_cast<uint4*>(codes + (w.values ? r.d * block + r.place : r.place * D + r.d));
    uint32_t four[4] = {0u, 0u, 0u, 0u};
    if (!empty && r.place < w.to) {
      if (old_places != 0u) {
        const uint4 old = *to;
        const uint32_t o[4] = {old.x, old.y, old.z, old.w}, olds = w.values ? old_places : 16u;
#pragma unroll
        for (uint32_t e = 0; e < 16u; ++e) {
          if (e < olds) x[n][e] = decode<KIND>(o[e / 4], static_cast<int>(e % 4)) * before;
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          four[j] = encode4<KIND>(x[n][4 * j], x[n][4 * j + 1], x[n][4 * j + 2], x[n][4 * j + 3], scale);
          if (!again && 4u * j < olds) {                   // codes that stay
            const uint32_t stay = olds - 4u * j, mask = stay < 4u ? (1u << 8u * stay) - 1u : ~0u;
            four[j] = (four[j] & ~mask) | (o[j] & mask);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) four[j] = encode4<KIND>(x[n][4 * j], x[n][4 * j + 1], x[n][4 * j + 2], x[n][4 * j + 3], scale);
      }
    }
    *to = uint4{four[0], four[1], four[2], four[3]};
  }
}

// Bound by memory: 2 bytes a row's element in, 8 or 4 out.  A workgroup takes the keys or the values of a head at 64 places that begin at
// a multiple of 64, so that pages of 16 places do not make a workgroup of 16 bytes a thread.  32768 rows of 4 heads of 256 as fp16, 201 MB: 33 us
// out of the last cache, 45 out of memory (a workgroup a page and a fp16 number a lane: 38 and 58).
constexpr uint32_t kReadPlaces = 64;
__device__ __forceinline__ uint32_t read_units(const PageSequence& q) { return (q.len - 1u) / kReadPlaces - (q.len - q.rows) / kReadPlaces + 1u; }

template <PageKind KIND, class Out>
__global__ __launch_bounds__(kPageThreads) void pages_read_kernel(PageBatch b, const uint8_t* __restrict__ kp, const uint8_t* __restrict__ vp,
                                                                  const float* __restrict__ ks, const float* __restrict__ vs, Out* __restrict__ k,
                                                                  Out* __restrict__ v) {
  __shared__ uint32_t page_of[4];
  __shared__ float scale_of[4];
  const uint32_t which = blockIdx.x % (2u * b.kv_heads), t = threadIdx.x, D = b.head_dim;
  PageUnit u;
  if (!find_unit(b, blockIdx.x / (2u * b.kv_heads), [](const PageSequence& q) { return read_units(q); }, &u)) return;
  const bool values = which >= b.kv_heads;
  const uint32_t kv = values ? which - b.kv_heads : which, past = u.seq.len - u.seq.rows, base = (past / kReadPlaces + u.at) * kReadPlaces;
  const uint32_t from = past > base ? past - base : 0u, to = u.seq.len - base < kReadPlaces ? u.seq.len - base : kReadPlaces;
  // Quarters of sixteen places, each in one page.  (Those behind the last position are the last one's, and not used.)
  if (t < 4u) {
    const uint32_t at = 16u * t < to ? base + 16u * t : u.seq.len - 1u, page = b.table[static_cast<uint64_t>(u.s) * b.width + (at >> b.log_block)];
    page_of[t] = page;
    scale_of[t] = page < b.pages ? (values ? vs : ks)[static_cast<uint64_t>(page) * b.kv_heads + kv] : 0.0f;
  }
  __syncthreads();
  const uint64_t wide = static_cast<uint64_t>(b.kv_heads) * D;
  Out* rows = (values ? v : k) + static_cast<uint64_t>(u.seq.first + (base + from - past)) * wide + kv * D;   // of place `from`
  const uint32_t block = 1u << b.log_block;
  auto head_of = [&](uint32_t quarter) {
    const uint32_t page = page_of[quarter];
    return (values ? vp : kp) + (static_cast<uint64_t>(page < b.pages ? page : 0u) * b.kv_heads + kv) * (static_cast<uint64_t>(block) * D);
  };
  // (A page that is not held has the scale 0 here; its codes may be a NaN's.)
  auto value = [&](uint32_t four, int i, float scale, bool held) {
    float x = held ? decode<KIND>(four, i) * scale : 0.0f;
    asm("" : "+v"(x));                                     // (an fp32 number before it is an fp16 one: no one operation for both)
    return static_cast<Out>(x);
  };
  if (!values) {
    constexpr uint32_t EACH = 16u / sizeof(Out);           // elements of a thread's sixteen bytes out
    typedef Out outs __attribute__((ext_vector_type(EACH)));
    const uint32_t runs = D / EACH, of_run = (1u << 20) / runs + 1u;      // (i < 64 * 64: i / runs by its product)
    const uint32_t end = to * runs;
    constexpr uint32_t AHEAD = 4;                          // loads on their way at once
    for (uint32_t i0 = t + from * runs; i0 < end; i0 += AHEAD * kPageThreads) {
      uint32_t four[AHEAD][EACH / 4];
#pragma unroll
      for (uint32_t n = 0; n < AHEAD; ++n) {
        const uint32_t i = i0 + n * kPageThreads < end ? i0 + n * kPageThreads : end - 1u;
        const uint32_t place = i * of_run >> 20, d = (i - place * runs) * EACH;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(head_of(place / 16u) + (((base + place) & (block - 1u)) * D + d));
#pragma unroll
        for (uint32_t j = 0; j < EACH / 4; ++j) four[n][j] = codes[j];
      }
#pragma unroll
      for (uint32_t n = 0; n < AHEAD; ++n) {
        const uint32_t i = i0 + n * kPageThreads;
        if (i >= end) break;
        const uint32_t place = i * of_run >> 20, d = (i - place * runs) * EACH, quarter = place / 16u;
        const float scale = scale_of[quarter];
        const bool held = page_of[quarter] < b.pages;
        outs x;
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) x[e] = value(four[n][e / 4], static_cast<int>(e % 4), scale, held);
        *reinterpret_cast<outs*>(rows + (place - from) * wide + d) = x;
      }
    }
    return;
  }
  // Sixteen places of two elements, which the next lane's follow in a row.
  const uint32_t pairs = D / 2u, of_pair = (1u << 20) / pairs + 1u, end = (to + 15u) / 16u * pairs;
  constexpr uint32_t AHEAD = 2;
  for (uint32_t i0 = t + from / 16u * pairs; i0 < end; i0 += AHEAD * kPageThreads) {
    uint4 run[AHEAD][2];
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) {
      const uint32_t i = i0 + n * kPageThreads < end ? i0 + n * kPageThreads : end - 1u;
      const uint32_t quarter = i * of_pair >> 20, d = (i - quarter * pairs) * 2u;
      const uint8_t* codes = head_of(quarter) + (d * block + ((base + quarter * 16u) & (block - 1u)));
      run[n][0] = load_u4(codes), run[n][1] = load_u4(codes + block);
    }
#pragma unroll
    for (uint32_t n = 0; n < AHEAD; ++n) {
      const uint32_t i = i0 + n * kPageThreads;
      if (i >= end) break;
      const uint32_t quarter = i * of_pair >> 20, d = (i - quarter * pairs) * 2u, place = quarter * 16u;
      const uint32_t r[2][4] = {{run[n][0].x, run[n][0].y, run[n][0].z, run[n][0].w}, {run[n][1].x, run[n][1].y, run[n][1].z, run[n][1].w}};
      const float scale = scale_of[quarter];
      const bool held = page_of[quarter] < b.pages;
      typedef Out out2 __attribute__((ext_vector_type(2)));
      Out* out = rows + static_cast<int64_t>(static_cast<int32_t>(place - from)) * static_cast<int64_t>(wide) + d;
      const bool whole = place >= from && place + 16u <= to;
#pragma unroll
      for (uint32_t e = 0; e < 16u; ++e) {
        if (whole || (place + e >= from && place + e < to)) {
          *reinterpret_cast<out2*>(out + e * wide) = out2{value(r[0][e / 4], static_cast<int>(e % 4), scale, held), value(r[1][e / 4], static_cast<int>(e % 4), scale, held)};
        }
      }
    }
  }
}

uint32_t workgroups(const PageCall& c) { return static_cast<uint32_t>(c.touched() * c.kv_heads * 2); }

}  // namespace

PageBatch page_batch(const PageCall& c, const uint32_t* table, const uint32_t* starts, const uint32_t* lens) {
  uint32_t log_block = 4;
  while ((uint64_t{1} << log_block) < c.block) ++log_block;
  return PageBatch{table, starts, lens, static_cast<uint32_t>(c.rows), static_cast<uint32_t>(c.sequences), static_cast<uint32_t>(c.pages),
                   static_cast<uint32_t>(c.width), static_cast<uint32_t>(c.rows), static_cast<uint32_t>(c.width * c.block),
                   static_cast<uint32_t>(c.kv_heads), static_cast<uint32_t>(c.head_dim), log_block};
}

hipError_t launch_pages_write(bool fp8, const PageWriteCall& c, const float* k, const float* v, const uint32_t* table, const uint32_t* starts,
                              const uint32_t* lens, uint8_t* kp, uint8_t* vp, float* ks, float* vs, hipStream_t stream) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(workgroups(c.page)), dim3(kPageThreads), 0, stream, page_batch(c.page, table, starts, lens), k, v, c.k_stride, c.v_stride,
                       kp, vp, ks, vs);
  };
  const uint64_t runs = c.page.block * c.page.head_dim / 16;      // of a page: at most 2048
  auto with = [&](auto items) {
    constexpr int N = decltype(items)::value;
    fp8 ? go(pages_write_kernel<PageKind::Fp8, N>) : go(pages_write_kernel<PageKind::Q8, N>);
  };
  runs <= 256 ? with(std::integral_constant<int, 1>{}) : runs <= 512 ? with(std::integral_constant<int, 2>{})
  : runs <= 1024 ? with(std::integral_constant<int, 4>{}) : with(std::integral_constant<int, 8>{});
  return hipGetLastError();
}

hipError_t launch_pages_read(bool fp8, const PageReadCall& c, const uint8_t* kp, const uint8_t* vp, const float* ks, const float* vs, const uint32_t* table,
                             const uint32_t* starts, const uint32_t* lens, void* k, void* v, hipStream_t stream) {
  // (a sequence's rows lie in at most two runs of 64 places more than they fill)
  const uint64_t some = c.page.rows / kReadPlaces + 2 * c.page.sequences, units = some < c.page.rows ? some : c.page.rows;
  auto go = [&](auto kernel, auto* as) {
    using Out = std::remove_pointer_t<decltype(as)>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(units * c.page.kv_heads * 2)), dim3(kPageThreads), 0, stream, page_batch(c.page, table, starts, lens), kp, vp, ks, vs,
                       static_cast<Out*>(k), static_cast<Out*>(v));
  };
  float* f32 = nullptr;
  _Float16* f16 = nullptr;
  if (c.f16) fp8 ? go(pages_read_kernel<PageKind::Fp8, _Float16>, f16) : go(pages_read_kernel<PageKind::Q8, _Float16>, f16);
  else fp8 ? go(pages_read_kernel<PageKind::Fp8, float>, f32) : go(pages_read_kernel<PageKind::Q8, float>, f32);
  return hipGetLastError();
}

}  // namespace qmm
