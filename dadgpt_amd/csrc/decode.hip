// KV-cache decode attention for gfx950: one query token per (sequence, head) against a
// ragged cache. Replaces the per-head GEMV chain of model_forward_cached
// (src/model.cpp:758-790: q K^T, *scale, softmax, P V) with one launch for all sequences and
// heads. Decode is a GEMV: it is bound by HBM, so it uses no MFMA.
//
// Cache layout [n_seq, H, max_len, D] (for n_seq = 1 this is the reference's per-layer
// [H, max_len, d_head] cache, src/model.cpp:659-675); only the first lens[s] rows are read.
//
// Work split. A cache (one sequence and head) is cut into chunks of C = 8*KW keys, one 8-wave
// workgroup per chunk; wave w owns keys [chunk*C + w*KW, chunk*C + (w+1)*KW). Every 16-byte
// load instruction of a wave covers whole key rows (bf16 D=64: 8 lanes x 16 B per row, 8 rows
// per instruction, a contiguous 1 KiB), all K and V loads of a wave are issued before any
// arithmetic, and they carry the non-temporal hint (the cache is streamed once). bf16 scores
// are v_dot2_f32_bf16 on the packed q and K words, so neither side is unpacked; the
// reductions across lanes use DPP and v_permlane16/32_swap (lanes.hpp), not LDS round trips. The 8 waves
// merge (max, sum, o) in LDS with the logsumexp rule. Chunks are small enough that the work
// of a long cache spreads over several CUs: one CU streaming a whole 1024-key cache alone was
// the tail of the launch.
//
// The grid runs over caches fastest, so consecutive workgroups (dealt round-robin to the 8
// XCDs) hold the same chunk index of different caches, and the chunks past a short cache's
// length (which exit at once) do not pile up on one XCD.
//
// A cache that fits one chunk is written directly. A longer one merges inside the same kernel:
// each chunk publishes an fp32 partial (max in log2 units, sum, unnormalised o) and counts
// itself on a per-cache counter; the chunk that arrives last merges all partials, writes the
// output and rearms the counter to zero.
//
// Ordering of that merge. The partials and the counter move only through agent-scope relaxed
// atomic accesses, and the rules that make this correct are those of the AMDGPU memory model
// for gfx942/gfx950 (LLVM AMDGPUUsage, "Memory Model GFX942"): a monotonic agent-scope atomic
// store, load or read-modify-write is a global_store / global_load / global_atomic with sc1 = 1,
// which is coherent across the 8 XCDs on its own (it bypasses the XCD-local L2), and
// s_waitcnt vmcnt(0) after a store waits for the store to complete. The publish sequence
// (sc1 stores, vmcnt(0), sc1 atomic increment; the last arriver reads with sc1 loads) is
// the compiler's agent-scope release / acquire sequence without its L2 writeback and
// invalidate, which only plain (non-sc1) accesses need. A release fence here writes back the
// whole L2, which made the first fence-based version of this kernel 17x slower. Other targets
// compile the standard release / acquire pair (DADGPT_DECODE_SC1_COHERENT, decode.hpp).
#include <mutex>

#include "common.hpp"
#include "decode.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace dadgpt {
namespace {

constexpr int kWaves = 8;         // waves per workgroup (one chunk)
constexpr int kLoadsPerWave = 8;  // 16-byte loads per lane and tensor

// Keys per wave: kLoadsPerWave wave-wide loads of 64 x 16 B, each covering whole key rows.
// bf16: 64 keys (D=64) or 128 (D=32); fp32: 32 or 64.
template <typename T, int D>
__host__ __device__ constexpr int keys_per_wave() {
  return kLoadsPerWave * 64 / (D / Elem<T>::kPer16B);
}
template <typename T, int D>
__host__ __device__ constexpr int chunk_keys() {
  return kWaves * keys_per_wave<T, D>();
}

// WIN: the keys are those the cache's last row sees through a sliding window with sinks, counted
// without the gap between the two (VisibleKeys): the chunks then cover min(len, window + sinks)
// keys, and only a key's row differs (8 x 12 fp32 caches of up to 16384 rows, window 4096, 176 MB:
// 31 us, 5.7 TB/s). A window of the whole cache runs it too: it takes as long as the plain kernel
// there (32 x 12 ragged bf16 caches of 1024 rows 13.6 us and 13.6, 8 x 12 fp32 of 32768 194 and 194),
// gives its bits, and a NaN key makes its row NaN for every window (the plain kernel answers 0 in an
// unsplit cache).
template <typename T, int D, bool WIN>
__global__ __launch_bounds__(64 * kWaves) void decode_kernel(
    T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ kc,
    const T* __restrict__ vc, const int* __restrict__ lens, int H, int max_len,
    float scale_log2, float* __restrict__ part, unsigned* __restrict__ counter, int n_chunk,
    const WindowArg<WIN> win) {
  constexpr int EPL = Elem<T>::kPer16B;       // elements per 16-byte load
  constexpr int KW = keys_per_wave<T, D>();   // keys per wave
  constexpr int C = chunk_keys<T, D>();       // keys per workgroup
  constexpr int LPR = D / EPL;                // lanes per key row
  constexpr int KPL = 64 / LPR;               // key rows per wave-wide load
  constexpr int NLD = kLoadsPerWave;          // loads per wave, per tensor
  __shared__ MergeLds<D, kWaves> sm;

  const int seq = blockIdx.x / H, head = blockIdx.x % H, chunk = blockIdx.y;
  const VisibleKeys<WIN> keys(clamp_len(lens[seq], max_len), win);
  const int L = keys.count;
  const int nch = (L + C - 1) / C;
  // Chunks past the length do nothing; chunk 0 of an empty cache still writes the zero output.
  if (chunk >= (nch > 1 ? nch : 1)) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane % LPR, grp = lane / LPR;
  const size_t hrow = (size_t)seq * H + head;
  const T* kh = kc + hrow * max_len * D + sub * EPL;
  const T* vh = vc + hrow * max_len * D + sub * EPL;
  const int key0 = chunk * C + wave * KW;

  float mx = neg_inf(), lsum = 0.f;
  float o[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) o[e] = 0.f;

  if (key0 < L) {  // wave-uniform: waves past the length skip their loads
    // q first (it is small and read by every chunk of the cache), kept packed.
    const u32x4 qw = ld_g128u(q + hrow * D + sub * EPL);
    // Rows past the length load row L-1 instead (valid, since key0 < L) and are masked out
    // below: the loads stay unconditional, so the compiler issues all of them back to back.
    u32x4 kr[NLD], vr[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int key = min(key0 + i * KPL + grp, L - 1);
      kr[i] = ld_stream(kh + (size_t)keys.row(key) * D);
    }
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int key = min(key0 + i * KPL + grp, L - 1);
      vr[i] = ld_stream(vh + (size_t)keys.row(key) * D);
    }
    // Keep the scheduler from sinking loads towards their uses: all of them stay in flight.
    __builtin_amdgcn_sched_barrier(0);

    // score of key key0 + i*KPL + grp: every lane of a row group ends with the full dot
    float s[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float acc = lanes::group_sum<LPR>(Elem<T>::dot(qw, kr[i]));
      const int key = key0 + i * KPL + grp;
      s[i] = key < L ? acc * scale_log2 : neg_inf();
      mx = fmaxf(mx, s[i]);
    }
    mx = lanes::wave_max_of_groups<LPR>(mx);  // uniform within each row group already
    // where every score is -inf, 0 stands in for the maximum: the keys' terms are 0
    const float base = mx == neg_inf() ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const float p = fast_exp2(s[i] - base);  // exactly 0 for masked rows
      lsum += p;
      float vf[EPL];
      Elem<T>::unpack(vr[i], vf);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = fmaf(p, vf[e], o[e]);
    }
    // sum over the row groups: lanes with the same column slice (lane % LPR) are partners
    if constexpr (LPR < 8) {
      lsum += __shfl_xor(lsum, LPR, 64);
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] += __shfl_xor(o[e], LPR, 64);
    }
    constexpr int K0 = LPR < 8 ? 8 : LPR;
    lsum = lanes::sum_across<K0>(lsum);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = lanes::sum_across<K0>(o[e]);
  }
  merge_chunks<!WIN, T, D, kWaves>(sm, out + hrow * D, o, mx, lsum, wave, lane, grp == 0,
                                   sub * EPL, chunk, nch, part + hrow * n_chunk * (D + 2),
                                   counter + hrow);
}

template <typename T, int D>
int n_chunk_for(int max_len) {
  return (max_len + chunk_keys<T, D>() - 1) / chunk_keys<T, D>();
}

template <typename T, int D>
hipError_t launch_decode_d(T* out, const T* q, const T* kc, const T* vc, const int* lens,
                           int n_seq, int H, int max_len, float scale, void* workspace,
                           size_t workspace_bytes, const Window* window, hipStream_t stream) {
  const int nc = n_chunk_for<T, D>(window ? visible_keys(max_len, *window) : max_len);
  float* part = nullptr;
  unsigned* counter = nullptr;
  if (nc > 1) {
    // the caller checked workspace_bytes >= decode_workspace_bytes(), which bounds both regions
    const size_t at = (workspace_bytes - partial_bytes(n_seq, H, nc, D)) & ~(size_t)15;
    counter = static_cast<unsigned*>(workspace);
    part = reinterpret_cast<float*>(static_cast<char*>(workspace) + at);
  }
  if (window != nullptr)
    decode_kernel<T, D, true><<<dim3(n_seq * H, nc), 64 * kWaves, 0, stream>>>(
        out, q, kc, vc, lens, H, max_len, scale * kLog2e, part, counter, nc, {*window});
  else
    decode_kernel<T, D, false><<<dim3(n_seq * H, nc), 64 * kWaves, 0, stream>>>(
        out, q, kc, vc, lens, H, max_len, scale * kLog2e, part, counter, nc, {});
  return hipGetLastError();
}

template <typename T>
hipError_t launch_decode_t(T* out, const T* q, const T* kc, const T* vc, const int* lens,
                           int n_seq, int H, int max_len, int D, float scale, void* workspace,
                           size_t workspace_bytes, const Window* window, hipStream_t stream) {
  if (D == 64)
    return launch_decode_d<T, 64>(out, q, kc, vc, lens, n_seq, H, max_len, scale, workspace,
                                  workspace_bytes, window, stream);
  if (D == 32)
    return launch_decode_d<T, 32>(out, q, kc, vc, lens, n_seq, H, max_len, scale, workspace,
                                  workspace_bytes, window, stream);
  return hipErrorInvalidValue;
}

// Scratch of the allocation-free entry point: it stands in for a caller's workspace (same
// layout: counters at the start, partials against the end) and lives as long as the code
// object, one copy per device. In host code `scratch` names a host-side shadow, not device
// memory: only the address hipGetSymbolAddress returns for the current device may reach a
// kernel or a copy.
static __device__ __align__(256) unsigned char scratch[kDecodeScratchBytes];

__global__ void zero_words_kernel(unsigned* p, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (size_t)gridDim.x * blockDim.x)
    p[i] = 0u;
}

}  // namespace

hipError_t decode_scratch(void** ptr, hipStream_t stream) {
  constexpr int kMaxDevices = 64;
  static std::mutex mu;
  static void* addr[kMaxDevices] = {};
  int dev = -1;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (addr[dev] == nullptr) {
    void* p = nullptr;
    if (hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)); e != hipSuccess) return e;
    if (p == nullptr) return hipErrorInvalidSymbol;
    // The arrival counters must start at zero (every call leaves them at zero again). A fill
    // kernel, not a memset node, so that a first call made under graph capture replays right.
    zero_words_kernel<<<256, 256, 0, stream>>>(static_cast<unsigned*>(p),
                                               kDecodeScratchBytes / sizeof(unsigned));
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    addr[dev] = p;
  }
  *ptr = addr[dev];
  return hipSuccess;
}

size_t decode_workspace_bytes(int n_seq, int H, int max_len, int D) {
  // fp32 chunks are shorter, so the fp32 chunk count bounds the bf16 one: the size returned
  // serves both element types.
  const int nc = D == 64 ? n_chunk_for<float, 64>(max_len) : n_chunk_for<float, 32>(max_len);
  if (nc == 1) return 0;
  return counter_bytes(n_seq, H) + partial_bytes(n_seq, H, nc, D);
}

hipError_t launch_decode_bf16(bf16* out, const bf16* q, const bf16* k_cache,
                              const bf16* v_cache, const int* lens, int n_seq, int H,
                              int max_len, int D, float scale, void* workspace,
                              size_t workspace_bytes, hipStream_t stream,
                              const Window* window) {
  return launch_decode_t<bf16>(out, q, k_cache, v_cache, lens, n_seq, H, max_len, D, scale,
                               workspace, workspace_bytes, window, stream);
}

hipError_t launch_decode_f32(float* out, const float* q, const float* k_cache,
                             const float* v_cache, const int* lens, int n_seq, int H,
                             int max_len, int D, float scale, void* workspace,
                             size_t workspace_bytes, hipStream_t stream,
                             const Window* window) {
  return launch_decode_t<float>(out, q, k_cache, v_cache, lens, n_seq, H, max_len, D, scale,
                                workspace, workspace_bytes, window, stream);
}

}  // namespace dadgpt
