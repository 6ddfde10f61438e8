// C entry points of a decode step whose requests share their beginnings: the checks of their arguments, which need no device.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "beam_step.h"
#include "errors.h"

using namespace b200;

namespace {

int refuse(const char* op, const char* why) {
  set_error("%s: %s", op, why);
  return B200_ERR_INVALID;
}
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
int launched(const char* op, int rc) { return rc ? cuda_fail(op, rc) : 0; }

}  // namespace

extern "C" {

int b200_op_norm_rope_kvwrite(const b200_norm_rope_args* a, void* stream) {
  const char* op = "b200_op_norm_rope_kvwrite";
  if (!a || a->T < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->num_pages < 0) return refuse(op, "bad sizes");
  if (a->q_heads > 4096 || a->kv_heads > 4096) return refuse(op, "more than 4096 heads");
  if (a->dims < 0 || a->dims > 128 || a->dims % 2) return refuse(op, "an even number of up to 128 values of a head is turned");
  if ((a->q_heads + 2 * a->kv_heads) * 128 > a->ldx || (a->q_heads && a->q_heads * 128 > a->ldo) || a->ldx % 8 || a->ldo % 8) return refuse(op, "rows of qkv and out are whole heads, a multiple of 8 apart");
  if ((a->q_norm_ld && a->q_norm_ld != 128) || (a->k_norm_ld && a->k_norm_ld != 128)) return refuse(op, "a norm has 128 weights, or 128 for each head");
  if (!(a->eps >= 0.f && a->eps < 1e30f) || !(a->gain > -1e30f && a->gain < 1e30f)) return refuse(op, "eps is no number of 0 and more, or gain is none");
  if (!a->T || !(a->q_heads + a->kv_heads)) return 0;
  if (!a->qkv || !a->positions || !a->slots || (a->dims && !a->freqs) || (a->q_heads && !a->out) || (a->kv_heads && a->num_pages && !a->kv_layer)) return refuse(op, "a buffer is missing");
  if (!aligned(a->qkv, 16) || !aligned(a->out, 16) || !aligned(a->kv_layer, 16) || !aligned(a->q_norm, a->norm_f32 ? 16 : 8) || !aligned(a->k_norm, a->norm_f32 ? 16 : 8))
    return refuse(op, "qkv, out, the cache and fp32 norms are 16-byte aligned, bf16 norms 8-byte");
  if (a->out == a->qkv && a->ldo != a->ldx && a->T > 1) return refuse(op, "queries kept in place have the rows of qkv");
  if (int rc = require_device()) return rc;
  return launched(op, norm_rope_kv_write(*a, static_cast<cudaStream_t>(stream)));
}

static int shared_sizes(const b200_shared_attn_args* a, const char* op) {
  if (!a || a->S < 0 || a->T < 0 || a->G < 0 || a->max_blocks < 0 || a->ld_tables < a->max_blocks || a->max_rows < 0 || a->max_ctx < 0 || a->num_pages < 0) return refuse(op, "bad sizes");
  const int group = a->kv_heads > 0 && a->q_heads > 0 && a->q_heads % a->kv_heads == 0 ? a->q_heads / a->kv_heads : 0;
  if (group != 1 && group != 2 && group != 4 && group != 8) return refuse(op, "a key head serves 1, 2, 4 or 8 heads");
  if (a->S > 65534 || a->G > 65534 || a->kv_heads > 4096) return refuse(op, "too many requests, groups or heads for a launch");
  if (a->max_blocks > INT_MAX / tree::kPage || a->num_pages >= INT_MAX / (32ll * a->kv_heads)) return refuse(op, "positions or cache rows pass 32 bits");
  if (static_cast<int64_t>(a->q_heads) * 128 > a->ldq || static_cast<int64_t>(a->q_heads) * 128 > a->ldo || a->ldq % 8 || a->ldo % 8) return refuse(op, "rows of q and out are whole heads, a multiple of 8 apart");
  if (!(a->scale > 0.f && a->scale < 1e30f)) return refuse(op, "scale is no number above 0 and below 1e30");      // a row's maximum is looked for ahead of the scale
  if (a->T > INT_MAX / 8) return refuse(op, "too many rows");
  if (!beam::costs_fit(*a, false) && !beam::costs_fit(*a, true)) return refuse(op, "the pages of all requests pass 32 bits");
  return 0;
}

int64_t b200_op_paged_attn_shared_workspace(const b200_shared_attn_args* a) {
  if (int rc = shared_sizes(a, "b200_op_paged_attn_shared_workspace")) return rc;
  return a->S && a->T && a->max_rows ? shared_attention_workspace(*a) : 0;
}

int b200_op_paged_attn_shared(const b200_shared_attn_args* a, void* stream) {
  const char* op = "b200_op_paged_attn_shared";
  if (int rc = shared_sizes(a, op)) return rc;
  if (!a->T || !a->q_heads) return 0;
  if (!a->out || !aligned(a->out, 16)) return refuse(op, "out is missing or not 16-byte aligned");
  if (!a->S || !a->max_rows) {      // no row is anybody's
    if (!a->zero_rest) return 0;
    if (int rc = require_device()) return rc;
    return launched(op, cudaMemset2DAsync(a->out, a->ldo * 2ll, 0, a->q_heads * 256ll, a->T, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : -2);
  }
  if (!a->q || !a->kv_layer || !a->starts || !a->ctx || (a->max_blocks && !a->block_tables) || !a->num_pages || (a->G && (!a->group_starts || !a->shared))) return refuse(op, "a buffer is missing");
  if (!aligned(a->q, 16) || !aligned(a->kv_layer, 256)) return refuse(op, "q is 16-byte aligned, the cache is 256-byte aligned");
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < shared_attention_workspace(*a)) return refuse(op, "the workspace is missing, too small or not 16-byte aligned");
  if (int rc = require_device()) return rc;
  int* mark = nullptr;
  if (int rc = op_mark(&mark)) return rc;
  return launched(op, paged_attention_shared(*a, mark, static_cast<cudaStream_t>(stream)));
}

static int select_sizes(const b200_beam_select_args* a, const char* op) {
  if (!a || a->S < 0 || a->V < 1 || a->ld < a->V || a->num_ends < 0) return refuse(op, "bad sizes");
  if (a->beams < 1 || a->beams > beam::kMaxBeams) return refuse(op, "1 to 32 beams");
  if (a->k < 1 || a->k > beam::kMaxFound) return refuse(op, "1 to 64 candidates");
  if (a->V > beam::kMaxVocab) return refuse(op, "more than 393216 tokens");
  if (a->num_ends > beam::kMaxEnds) return refuse(op, "more than 1024 tokens that end a text");
  if (a->S > INT_MAX / (64 * a->beams)) return refuse(op, "too many requests for a launch");
  return 0;
}

int64_t b200_op_beam_select_workspace(const b200_beam_select_args* a) {
  if (int rc = select_sizes(a, "b200_op_beam_select_workspace")) return rc;
  return a->S ? beam_select_workspace(*a) : 0;
}

int b200_op_beam_select(const b200_beam_select_args* a, void* stream) {
  const char* op = "b200_op_beam_select";
  if (int rc = select_sizes(a, op)) return rc;
  if (!a->S) return 0;
  if (!a->logits || !a->scores || (a->num_ends && !a->ends) || !a->parents || !a->tokens || !a->new_scores || !a->found_parents || !a->found_tokens || !a->found_scores)
    return refuse(op, "a buffer is missing");
  if (!aligned(a->logits, a->logits_f32 ? 4 : 2)) return refuse(op, "logits lie off their type's alignment");
  if (a->new_scores == a->scores) return refuse(op, "new scores have a buffer of their own");
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < beam_select_workspace(*a)) return refuse(op, "the workspace is missing, too small or not 16-byte aligned");
  if (int rc = require_device()) return rc;
  int* mark = nullptr;
  if (int rc = op_mark(&mark)) return rc;
  return launched(op, beam_select(*a, mark, static_cast<cudaStream_t>(stream)));
}

int b200_op_beam_reorder(const b200_beam_reorder_args* a, void* stream) {
  const char* op = "b200_op_beam_reorder";
  if (!a || a->S < 0 || a->max_blocks < 0 || a->ld_tables < a->max_blocks || a->ld_tables_out < a->max_blocks || a->layers < 0 || a->num_pages < 0 || a->room < 0) return refuse(op, "bad sizes");
  if (a->beams < 1 || a->beams > beam::kMaxBeams) return refuse(op, "1 to 32 beams");
  if (a->max_blocks > INT_MAX / tree::kPage) return refuse(op, "positions pass 32 bits");
  if (a->S > INT_MAX / beam::kMaxBeams) return refuse(op, "too many requests for a launch");
  if (a->layers && (!a->kv || a->kv_heads < 1 || a->kv_heads > 4096 || a->layer_stride % 8 || a->layer_stride / 4096 < a->num_pages * (a->layers > 1) * a->kv_heads))
    return refuse(op, "layers of the cache are missing, overlap or lie a number of elements apart that 8 does not divide");
  if (a->layers && !aligned(a->kv, 16)) return refuse(op, "the cache is 16-byte aligned");
  if (a->texts && (a->ld_texts < a->room || a->ld_texts_out < a->room)) return refuse(op, "texts have less room than they say");
  if (!a->S) return 0;
  if (!a->parents || !a->ctx || !a->shared || (a->max_blocks && (!a->block_tables || !a->tables_out || !a->released)) || (a->texts && (!a->tokens || !a->texts_out || !a->text_lens || !a->text_lens_out)))
    return refuse(op, "a buffer is missing");
  if ((a->max_blocks && a->tables_out == a->block_tables) || (a->texts && (a->texts_out == a->texts || a->text_lens_out == a->text_lens))) return refuse(op, "what comes out has buffers of its own");
  if (int rc = require_device()) return rc;
  return launched(op, beam_reorder(*a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
