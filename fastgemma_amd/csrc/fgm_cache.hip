// fgm_cache.hip -- bounded KV caches on gfx950: which slots a cache keeps
// (select_kernel) and the move of chosen slots to the front (move_kernel).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fgm_common.h"
#include "fgm_kernels.h"

namespace {

// ----------------------------------------------------------------- select
// Order-preserving key of a weight: NaN as minus infinity, both zeros alike.
FGM_DEV uint32_t weight_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// grid (sequences), 1024 threads.  Of the n slots the first `sink` and the last
// `recent` stay; of the others, [lo, hi), the `need` with the largest keys.
// Radix select over the bits 31..21, 20..10 and 9..0 of the key: each pass counts
// the keys that agree with the digits found so far by their next digit, and the
// digit is where the running count from the top reaches what is still needed.  A
// pass ends the search when the keys of its digit are all needed, or one is left.
// Wave w holds the slots of its own stretch in registers, NV a lane, so that the
// weights are read once and the kept slots come out in ascending order with one
// count per wave (NV = 0: stretches of any length, read again in every pass).
// Bound by the latency of one workgroup's chain, not by the 4 bytes a slot: 16
// sequences x 32000 slots -> 4096 20.0 us (load 5, first pass 4, the others 2.8
// each, count and write 3; 47 us as four 8-bit passes over memory), 1100 -> 512
// 5.6 us.  The first pass's LDS atomics meet in the few bins of the exponents.
template <int NV>
__global__ __launch_bounds__(1024) void select_kernel(const SelectBatch b) {
  constexpr int BINS = 2048;
  __shared__ int hist[BINS];
  __shared__ int s_part[16], s_digit, s_k, s_count, wgt[16], weq[16];
  const SelectProb p = b.p[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const int n = p.n, budget = b.budget;
  if (n <= budget) {
    for (int i = tid; i < budget; i += 1024) p.keep[i] = i < n ? i : -1;
    return;
  }
  const int lo = b.sink, hi = n - b.recent, need = budget - b.sink - b.recent;
  for (int i = tid; i < lo; i += 1024) p.keep[i] = i;
  for (int i = tid; i < b.recent; i += 1024) p.keep[budget - b.recent + i] = hi + i;
  if (need == 0) return;
  // wave w's stretch [first, last), a multiple of 64 slots long but for the end
  const int seg = (hi - lo + 1023) / 1024 * 64;
  const int first = min(lo + w * seg, hi), last = min(first + seg, hi);
  uint32_t kept[NV ? NV : 1];
  const __amdgpu_buffer_rsrc_t rm = make_rsrc(p.mass, NV ? 4u * (uint32_t)last : 0);
#pragma unroll
  for (int v = 0; v < NV; v++) kept[v] = buf_load_b32(rm, 4u * (uint32_t)(first + 64 * v + lane), 0);
#pragma unroll
  for (int v = 0; v < NV; v++) kept[v] = weight_key(__uint_as_float(kept[v]));
  // f(key, whether a slot is there) for the lane's slots, in order
  auto each = [&](auto&& f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; v++)
        if (first + 64 * v < last) f(kept[v], first + 64 * v + lane);
    } else {
      for (int i = first + lane; i - lane < last; i += 64) f(i < last ? weight_key(p.mass[i]) : 0u, i);
    }
  };
  // after a pass: keys whose bits from `shift` on are above `prefix` are kept, of
  // those at it k
  uint32_t prefix = 0;
  int k = need, shift = 32;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int bits = pass < 2 ? 11 : 10, next = shift - bits;
    hist[tid] = hist[tid + 1024] = 0;
    __syncthreads();
    each([&](uint32_t key, int i) {
      if (i < last && (pass == 0 || key >> shift == prefix))
        atomicAdd(&hist[(key >> next) & ((1 << bits) - 1)], 1);
    });
    __syncthreads();
    // thread t: the bins BINS - 1 - 2 t and below it; counts from the top
    const int top = BINS - 1 - 2 * tid, c0 = hist[top], c1 = hist[top - 1];
    int run = c0 + c1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(run, d, 64);
      if (lane >= d) run += o;
    }
    if (lane == 63) s_part[w] = run;
    __syncthreads();
    int before = run - c0 - c1;
    for (int j = 0; j < w; j++) before += s_part[j];
    if (before < k && before + c0 + c1 >= k) {
      const bool second = before + c0 < k;
      s_digit = second ? top - 1 : top;
      s_k = k - before - (second ? c0 : 0);
      s_count = second ? c1 : c0;
    }
    __syncthreads();
    prefix = prefix << bits | (uint32_t)s_digit, k = s_k, shift = next;
    if (k == s_count) break;  // all of them
  }
  // kept: keys from `thr` on, and of those at `tie` the first k
  const bool ties = k != s_count;
  const uint32_t tie = prefix, thr = ties ? prefix + 1 : prefix << shift;  // no key is all ones
  int gt = 0, eq = 0;
  each([&](uint32_t key, int i) {
    gt += i < last && key >= thr;
    eq += ties && i < last && key == tie;
  });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) gt += __shfl_xor(gt, d, 64), eq += __shfl_xor(eq, d, 64);
  if (lane == 0) wgt[w] = gt, weq[w] = eq;
  __syncthreads();
  int at = lo, eqs = 0;  // kept slots and ties before this one
  for (int j = 0; j < w; j++) at += wgt[j], eqs += weq[j];
  at += min(eqs, k);
  each([&](uint32_t key, int i) {
    bool take = i < last && key >= thr;
    if (ties) {
      const unsigned long long E = __ballot(i < last && key == tie);
      if (E) {
        const int e = eqs + __builtin_amdgcn_mbcnt_hi((uint32_t)(E >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)E, 0));
        take |= (E >> lane & 1) && e < k;
        eqs += __builtin_popcountll(E);
      }
    }
    const unsigned long long K = __ballot(take);
    if (take) p.keep[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(K >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)K, 0))] = i;
    at += __builtin_popcountll(K);
  });
}

// ------------------------------------------------------------------- move
// Slot of the j-th position from slot0 on.
FGM_DEV int ring_slot(int slot0, int j, int ring) {
  const int s = slot0 + j;  // below 2^31: capacities are at most 2^30
  return ring && s >= ring ? s - ring : s;
}

// grid (slices, problems, chunks), 1024 threads.  A slice is KS bytes of every K
// row, VS dims of every V group, or the scales.  In place one workgroup takes a
// slice's whole list, in batches that are read whole before they are written:
// the list ascends, so index[j] >= j, and what a batch writes no later batch
// reads.  Into another cache the chunks go to workgroups of their own.  V lies in
// groups of four slots, so a moved slot's byte is picked out of each dword of its
// group: four 16-byte reads a 16-byte write.  8 caches of 8192 slots x 512 cut to
// 2048: 13.2 us for 17 MB moved and about 42 MB read (28.7 us with V slices of 64
// dims, half the workgroups, and the list read from memory).
// VEC: 16-byte accesses (rows a multiple of 16 bytes at 16-byte addresses).
constexpr int MOVE_LIST = 4096;
// bytes of a K row and dims of a V group in a slice
constexpr int KS = 64, VS = 32;

template <int T, bool IN_PLACE, bool VEC>
__global__ __launch_bounds__(T) void move_kernel(const MoveBatch b) {
  __shared__ int s_end, s_list[MOVE_LIST];
  const MoveProb p = b.p[blockIdx.y];
  const int tid = threadIdx.x, row = b.row;
  // the list ends at the first entry that does not ascend or lies outside; its
  // first entries, as source slots, stay in LDS
  if (tid == 0) s_end = p.count;
  __syncthreads();
  for (int j = tid; j < p.count; j += T) {
    const int x = p.index[j], y = j ? p.index[j - 1] : -1;
    if (x <= y || x >= p.limit) atomicMin(&s_end, j);
    else if (j < MOVE_LIST) s_list[j] = ring_slot(p.slot0, x, p.ring);
  }
  __syncthreads();
  const int n = s_end;
  const int kslices = (row + KS - 1) / KS, vslices = (row + VS - 1) / VS;
  const int z = blockIdx.z, nz = IN_PLACE ? 1 : (int)gridDim.z;
  auto from = [&](int j) { return j < MOVE_LIST ? s_list[j] : ring_slot(p.slot0, p.index[j], p.ring); };

  if ((int)blockIdx.x < kslices) {  // K: L lanes a row
    constexpr int L = VEC ? KS / 16 : KS, R = T / L, U = 8;
    typedef std::conditional_t<VEC, v4i, int8_t> unit;
    const int c = KS * blockIdx.x + (tid % L) * (int)sizeof(unit);
    const bool in = c < row;
    for (int j0 = z * R * U; j0 < n; j0 += nz * R * U) {
      unit x[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j = j0 + tid / L + R * u;
        if (in && j < n) x[u] = *(const unit*)(p.kc + (size_t)from(j) * row + c);
      }
      if (IN_PLACE) __syncthreads();
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j = j0 + tid / L + R * u;
        if (in && j < n) *(unit*)(p.kc_to + (size_t)ring_slot(p.slot0_to, j, p.ring_to) * row + c) = x[u];
      }
    }
  } else if ((int)blockIdx.x < kslices + vslices) {
    // V: groups of four destination slots, D dims a lane.  Where the run wraps in
    // its ring it has two stretches of groups.
    constexpr int D = VEC ? 4 : 1, L = VS / D, R = T / L, U = 4;
    const int c = VS * (blockIdx.x - kslices) + (tid % L) * D;
    const bool in = c < row;
    const int a0 = p.slot0_to, e0 = p.ring_to ? min(a0 + n, p.ring_to) : a0 + n, e1 = a0 + n - e0;
    const int g0 = a0 >> 2, ng0 = n ? ((e0 + 3) >> 2) - g0 : 0, ng = ng0 + ((e1 + 3) >> 2);
    for (int q0 = z * R * U; q0 < ng; q0 += nz * R * U) {
      uint32_t x[U][D];
      int grp[U], has[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int q = q0 + tid / L + R * u;
        const bool second = q >= ng0;
        grp[u] = second ? q - ng0 : g0 + q;
        has[u] = 0;
#pragma unroll
        for (int d = 0; d < D; d++) x[u][d] = 0;
        if (!in || q >= ng) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int s = 4 * grp[u] + i, j = second ? s + (e0 - a0) : s - a0;
          if (second ? s >= e1 : (s < a0 || s >= e0)) continue;
          has[u] |= 1 << i;
          const int f = from(j), sh = 8 * (f & 3);
          const int8_t* src = p.vt + ((size_t)(f >> 2) * row + c) * 4;
          if constexpr (VEC) {
            const v4i v = *(const v4i*)src;
#pragma unroll
            for (int d = 0; d < 4; d++) x[u][d] |= ((uint32_t)v[d] >> sh & 255u) << (8 * i);
          } else {
            x[u][0] |= (uint32_t)(uint8_t)src[f & 3] << (8 * i);
          }
        }
      }
      if (IN_PLACE) __syncthreads();
#pragma unroll
      for (int u = 0; u < U; u++) {
        int8_t* dst = p.vt_to + ((size_t)grp[u] * row + c) * 4;
        if constexpr (VEC) {
          if (has[u] == 15) {
            *(v4i*)dst = v4i{(int)x[u][0], (int)x[u][1], (int)x[u][2], (int)x[u][3]};
            continue;
          }
        }
        // a group that is part of the run: its other bytes belong to others
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (has[u] >> i & 1)
#pragma unroll
            for (int d = 0; d < D; d++) dst[4 * d + i] = (int8_t)(x[u][d] >> (8 * i));
      }
    }
  } else {
    for (int j0 = z * T; j0 < n; j0 += nz * T) {
      const int j = j0 + tid;
      float k = 0, v = 0, m = 0;
      if (j < n) {
        const int f = from(j);
        k = p.ks[f], v = p.vs[f];
        if (p.mass) m = p.mass[f];
      }
      if (IN_PLACE) __syncthreads();
      if (j < n) {
        const int t = ring_slot(p.slot0_to, j, p.ring_to);
        p.ks_to[t] = k, p.vs_to[t] = v;
        if (p.mass) p.mass_to[t] = m;
      }
    }
  }
}

}  // namespace

hipError_t fgm_launch_select(const SelectBatch& b, hipStream_t st) {
  if (b.count <= 0 || b.budget <= 0) return hipSuccess;
  int n = 0;
  for (int i = 0; i < b.count; i++) n = std::max(n, b.p[i].n);
  // the fewest registers that hold the longest sequence
  if (n <= 4 * 1024)
    hipLaunchKernelGGL(select_kernel<4>, dim3(b.count), dim3(1024), 0, st, b);
  else if (n <= 12 * 1024)
    hipLaunchKernelGGL(select_kernel<12>, dim3(b.count), dim3(1024), 0, st, b);
  else if (n <= 32 * 1024)
    hipLaunchKernelGGL(select_kernel<32>, dim3(b.count), dim3(1024), 0, st, b);
  else
    hipLaunchKernelGGL(select_kernel<0>, dim3(b.count), dim3(1024), 0, st, b);
  return hipGetLastError();
}

hipError_t fgm_launch_move(const MoveBatch& b, bool in_place, hipStream_t st) {
  if (b.count <= 0 || b.row <= 0 || b.max_count <= 0) return hipSuccess;
  bool vec = b.row % 16 == 0;
  for (int i = 0; i < b.count; i++)
    vec = vec && (((uintptr_t)b.p[i].kc | (uintptr_t)b.p[i].vt | (uintptr_t)b.p[i].kc_to |
                   (uintptr_t)b.p[i].vt_to) & 15) == 0;
  const int slices = (b.row + KS - 1) / KS + (b.row + VS - 1) / VS + 1;
  auto launch = [&](auto t, auto in, auto v) {
    constexpr int T = decltype(t)::value;
    const dim3 grid(slices, b.count, in_place ? 1 : std::min(64, (b.max_count + 2 * T - 1) / (2 * T)));
    hipLaunchKernelGGL((move_kernel<T, decltype(in)::value, decltype(v)::value>), grid, dim3(T), 0, st, b);
  };
  auto by_vec = [&](auto t, auto in) {
    if (vec) launch(t, in, std::true_type{});
    else launch(t, in, std::false_type{});
  };
  auto by_place = [&](auto t) {
    if (in_place) by_vec(t, std::true_type{});
    else by_vec(t, std::false_type{});
  };
  // accepted paths are tens of slots: four waves (16 lists of 26: 5.7 -> 4.8 us)
  if (b.max_count <= 256) by_place(std::integral_constant<int, 256>{});
  else by_place(std::integral_constant<int, 1024>{});
  return hipGetLastError();
}
