// Linear attention over ragged batches of chunks of tokens (prompts).
#include <cstring>
#include <new>

#include "mkv_linear.h"

using namespace mkv;

extern "C" int mkv_linear_extend(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                 const void *d_v, const float *d_log_decay, void *d_o, const int32_t *d_q_indptr,
                                 const int32_t *d_src_slots, const int32_t *d_dst_slots, int32_t num_seqs,
                                 int32_t num_tokens, int32_t max_q_len, float scale, uint32_t flags,
                                 void *d_workspace, uint64_t workspace_bytes, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  if (max_q_len < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "max_q_len < 0");
  LinArgs a;
  int rc = lin_args(p, layer, d_q, d_k, d_v, d_log_decay, d_o, d_src_slots, d_dst_slots, num_seqs, num_tokens, scale,
                    flags, a);
  if (rc) return rc;
  if (num_seqs && !d_q_indptr) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  a.q_indptr = d_q_indptr;
  DeviceGuard guard(p->device);
  return launch_recurrence(p, a, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int mkv_linear_extend_host(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                      const void *d_v, const float *d_log_decay, void *d_o, const int32_t *h_q_lens,
                                      const uint32_t *h_src_slots, const uint32_t *h_dst_slots, int32_t num_seqs,
                                      float scale, uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  int rc = check_state_slots(p, h_src_slots, h_dst_slots, num_seqs);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (!h_q_lens) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL lengths");
  int64_t tokens = 0;
  int32_t longest = 0;
  for (int32_t b = 0; b < num_seqs; b++) {
    if (h_q_lens[b] < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "q_len[%d] = %d < 0", b, h_q_lens[b]);
    tokens += h_q_lens[b];
    longest = std::max(longest, h_q_lens[b]);
  }
  if (tokens > INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "more than 2^31 - 1 tokens");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  if ((rc = refuse_capture(hs))) return rc;
  MetaSlot *sl = nullptr;
  const size_t B = (size_t)num_seqs;
  try {  // src | dst | q_indptr
    std::vector<int32_t> &st = p->stage_tmp;
    st.resize(3 * B + 1);
    std::memcpy(st.data(), h_src_slots ? h_src_slots : h_dst_slots, B * 4);
    std::memcpy(st.data() + B, h_dst_slots, B * 4);
    int32_t *ip = st.data() + 2 * B;
    ip[0] = 0;
    for (size_t b = 0; b < B; b++) ip[b + 1] = ip[b] + h_q_lens[b];
    if ((rc = stage_cached(p, p->extend_cache, st.data(), st.size(), hs, &sl))) return rc;
  } catch (const std::bad_alloc &) {
    return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  rc = mkv_linear_extend(pool, layer, d_q, d_k, d_v, d_log_decay, d_o, sl->d + 2 * B, sl->d, sl->d + B, num_seqs,
                         (int32_t)tokens, longest, scale, flags, nullptr, 0, stream);
  const int rr = meta_release(sl, hs);
  return rc ? rc : rr;
}
