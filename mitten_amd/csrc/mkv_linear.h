// Declarations shared by the linear-attention translation units.
#pragma once

#include <vector>

#include "mkv_internal.h"

namespace mkv {

// Pool of linear-attention states: f32 [layers][slots][value heads][k_dim][v_dim].
struct StatePool : MetaRing {
  mkv_state_desc desc;
  int device = 0;
  int cus = 0;  // compute units of the device
  float *data = nullptr;
  uint64_t bytes = 0;
  int64_t state_elems = 0;    // one slot of one layer
  uint32_t *d_err = nullptr;  // device error word
  void *ws = nullptr;         // workspace of split extend calls, allocated with the pool
  uint64_t ws_bytes = 0;
  hipEvent_t ws_done = nullptr;  // after the last eager call that used it
  bool ws_used = false;
  // Host arrays staged last by the step and extend entry points (every layer
  // of an engine step passes the same ones), scratch to assemble and to check
  // them in: mark[slot] = epoch of the call that last wrote the slot.
  StagedCache step_cache, extend_cache;
  std::vector<int32_t> stage_tmp;
  std::vector<uint32_t> mark, owner;
  uint32_t epoch = 0;
};

struct LinArgs {
  const void *q, *k;   // [tokens][Hk][DK]
  const void *v;       // [tokens][Hv][DV]
  const float *g;      // log decays: [tokens][Hv], or [Hv] when g_stride is 0
  void *o;             // [tokens][Hv][DV]
  float *states;       // the layer's plane: [slots][Hv][DK][DV]
  const int32_t *q_indptr;  // [B + 1], or null: one token per sequence
  const int32_t *src, *dst;
  uint32_t *d_err;
  int64_t nslots;
  int32_t B, Hk, Hv, DV, g_stride, num_tokens;
  float scale;
};

constexpr int32_t kMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads in one grid dimension

constexpr uint64_t kLinWorkspace = 64ull << 20;  // bytes of a state pool's own workspace

// One sequence's rows and slots; false: nothing to do (reported when `report`).
struct LinSeq {
  int32_t row0, n;
  int64_t src, dst;  // src < 0: starts from zero
};
__device__ __forceinline__ bool lin_seq(const LinArgs &a, int b, bool report, LinSeq &s) {
  s.row0 = b;
  s.n = 1;
  if (a.q_indptr) {
    s.row0 = a.q_indptr[b];
    const int64_t end = a.q_indptr[b + 1];
    if (s.row0 < 0 || end < s.row0 || end > a.num_tokens) {
      if (report) record_error(a.d_err, MKV_DEVERR_CTX);
      return false;
    }
    s.n = (int32_t)(end - s.row0);
  }
  s.src = a.src ? a.src[b] : a.dst[b];
  s.dst = a.dst[b];
  if (s.src < -1 || s.src >= a.nslots || s.dst < 0 || s.dst >= a.nslots) {
    if (report) record_error(a.d_err, MKV_DEVERR_SLOT);
    return false;
  }
  return true;
}

// ---- host side ------------------------------------------------------------------

// Checks what every linear entry point shares and fills the kernel arguments.
int lin_args(StatePool *p, int32_t layer, const void *d_q, const void *d_k, const void *d_v, const float *d_g,
             void *d_o, const int32_t *d_src, const int32_t *d_dst, int32_t num_seqs, int32_t num_tokens, float scale,
             uint32_t flags, LinArgs &a);
// Checks host slots: destinations inside the pool and distinct, sources
// inside it or MKV_STATE_NONE, and no source that another sequence writes.
int check_state_slots(StatePool *p, const uint32_t *src, const uint32_t *dst, int32_t n);
// Refuses a stream that is being captured (host metadata is staged in buffers
// that later calls reuse).
int refuse_capture(hipStream_t hs);

}  // namespace mkv
