// C entry points of a verification step of drafted tokens: the checks of their arguments, which need no device.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "errors.h"
#include "tree_step.h"

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

int b200_op_step_maps(const b200_step_maps_args* a, void* stream) {
  const char* op = "b200_op_step_maps";
  if (!a || a->S < 0 || a->T < 0 || a->max_blocks < 0 || a->num_free < 0 || a->ld_tables < a->max_blocks) return refuse(op, "bad sizes");
  if (a->S > tree::kMaxRequests) return refuse(op, "more than 8192 requests");
  if (a->T > tree::kMaxRows || a->num_free > tree::kMaxRows) return refuse(op, "more than 2^30 rows or pages");
  if (a->words < 0 || a->words > tree::kMaxWords) return refuse(op, "masks of more than 8 words");
  if (a->max_blocks > INT_MAX / tree::kPage) return refuse(op, "positions pass 32 bits");
  if (!a->starts || !a->cursor || !a->cursor_out || (a->S && (!a->ctx || !a->rows || !a->held || !a->held_out || !a->status)) || (a->T && (!a->positions || !a->slots || (a->words && !a->masks))) ||
      (a->num_free && !a->free_pages) || (a->S && a->max_blocks && !a->block_tables))
    return refuse(op, "a buffer is missing");
  if (int rc = require_device()) return rc;
  return launched(op, step_maps(*a, static_cast<cudaStream_t>(stream)));
}

static int attn_sizes(const b200_tree_attn_args* a, const char* op) {
  if (!a || a->S < 0 || a->T < 0 || a->max_blocks < 0 || a->ld_tables < a->max_blocks || a->max_tree < 0 || a->max_ctx < 0 || a->num_pages < 0) return refuse(op, "bad sizes");
  const int group = a->kv_heads > 0 && a->q_heads > 0 && a->q_heads % a->kv_heads == 0 ? a->q_heads / a->kv_heads : 0;
  if (group != 1 && group != 2 && group != 4 && group != 8) return refuse(op, "a key head serves 1, 2, 4 or 8 heads");
  if (a->S > 65534 || a->kv_heads > 4096) return refuse(op, "too many requests or heads for a launch");
  if (a->words < 0 || a->words > tree::kMaxWords || (a->masks && !a->words)) return refuse(op, "masks of 1 to 8 words");
  if (a->masks && a->max_tree > 32 * a->words) return refuse(op, "more rows of a request than its masks have bits");
  if (a->max_blocks > INT_MAX / tree::kPage || a->num_pages >= INT_MAX / (32ll * a->kv_heads)) return refuse(op, "positions or cache rows pass 32 bits");
  if (static_cast<int64_t>(a->q_heads) * 128 > a->ldq || static_cast<int64_t>(a->q_heads) * 128 > a->ldo || a->ldq % 8 || a->ldo % 8) return refuse(op, "rows of q and out are whole heads, a multiple of 8 apart");
  if (!(a->scale > 0.f && a->scale < 1e30f)) return refuse(op, "scale is no number above 0 and below 1e30");      // a row's maximum is looked for ahead of the scale
  const long long rows = static_cast<long long>(a->max_tree < a->T ? a->max_tree : a->T) * group;
  if ((rows + 127) / 128 * a->kv_heads > INT_MAX / 4 / (a->S + 1ll) / (a->max_blocks / 4 + 1)) return refuse(op, "the tiles of all requests pass 32 bits");
  return 0;
}

int64_t b200_op_paged_attn_tree_workspace(const b200_tree_attn_args* a) {
  if (int rc = attn_sizes(a, "b200_op_paged_attn_tree_workspace")) return rc;
  return a->S && a->T && a->max_tree ? tree_attention_workspace(*a) : 0;
}

int b200_op_paged_attn_tree(const b200_tree_attn_args* a, void* stream) {
  const char* op = "b200_op_paged_attn_tree";
  if (int rc = attn_sizes(a, op)) return rc;
  if (!a->T || !a->q_heads) return 0;
  if (!a->out || !aligned(a->out, 16)) return refuse(op, "out is missing or not 16-byte aligned");
  if (!a->S || !a->max_tree) {      // no row is anybody's
    if (!a->zero_rest) return 0;
    if (int rc = require_device()) return rc;
    return launched(op, cudaMemset2DAsync(a->out, a->ldo * 2ll, 0, a->q_heads * 256ll, a->T, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : -2);
  }
  if (!a->q || !a->kv_layer || !a->starts || !a->ctx || (a->max_blocks && !a->block_tables) || !a->num_pages) return refuse(op, "a buffer is missing");
  if (!aligned(a->q, 16) || !aligned(a->kv_layer, 256)) return refuse(op, "q is 16-byte aligned, the cache is 256-byte aligned");
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < tree_attention_workspace(*a)) return refuse(op, "the workspace is missing, too small or not 16-byte aligned");
  if (int rc = require_device()) return rc;
  int* mark = nullptr;
  if (int rc = op_mark(&mark)) return rc;
  return launched(op, paged_attention_tree(*a, mark, static_cast<cudaStream_t>(stream)));
}

int b200_op_constrain(const b200_constrain_args* a, void* stream) {
  const char* op = "b200_op_constrain";
  if (!a || a->S < 0 || a->T < 0 || a->V < 1 || a->ld < a->V || (a->out && a->ld_out < a->V)) return refuse(op, "bad sizes");
  if (a->V > 393216) return refuse(op, "more than 393216 tokens");
  if (a->S > 65534) return refuse(op, "more than 65534 requests");
  if (a->T > tree::kMaxRows || a->history_len > tree::kMaxSaid || a->bias_len > tree::kMaxRows) return refuse(op, "more than 2^30 rows or biases or 2^29 tokens of histories");
  if (!a->starts && a->S != a->T) return refuse(op, "without starts every row is a request");
  if (a->words < 0 || a->words > tree::kMaxWords || (a->masks && !a->words)) return refuse(op, "masks of 1 to 8 words");
  if (a->masks && !a->drafts) return refuse(op, "masks without drafts");
  if (a->drafts && !a->starts) return refuse(op, "drafts without starts");
  if (a->history && (!a->hist_starts || a->history_len < 0)) return refuse(op, "a history without its starts");
  if (a->bias_starts && a->bias_len && (!a->bias_ids || !a->bias_values)) return refuse(op, "biases without their tokens or values");
  if (a->bias_len < 0) return refuse(op, "bad sizes");
  if (a->allow && (a->ld_allow < (a->V + 31) / 32 || a->allow_count < 0)) return refuse(op, "rows of allow are narrower than the vocabulary");
  if (a->allow && !a->allow_rows && a->allow_count < a->T) return refuse(op, "fewer masks than rows");
  if (a->allow_rows && !a->allow) return refuse(op, "rows of masks that are not there");
  if (!a->T) return 0;
  if (!a->ids && !a->out) return refuse(op, "neither choices nor logits asked for");
  if (!a->S) {
    if (!a->ids) return 0;
    if (int rc = require_device()) return rc;
    return launched(op, cudaMemsetAsync(a->ids, 0xff, a->T * 4ll, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : -2);      // no row is anybody's: -1
  }
  if (!a->logits) return refuse(op, "a buffer is missing");
  if (!aligned(a->logits, a->logits_f32 ? 4 : 2) || !aligned(a->out, a->out_f32 ? 4 : 2)) return refuse(op, "logits lie off their type's alignment");
  if (a->out == a->logits && (a->ld_out != a->ld || !a->out_f32 != !a->logits_f32)) return refuse(op, "logits kept in place have their type and rows");
  if (int rc = require_device()) return rc;
  int* mark = nullptr;
  if (int rc = op_mark(&mark)) return rc;
  return launched(op, constrain(*a, mark, static_cast<cudaStream_t>(stream)));
}

int b200_op_tree_accept(const b200_tree_accept_args* a, void* stream) {
  const char* op = "b200_op_tree_accept";
  if (!a || a->S < 0 || a->T < 0 || a->max_blocks < 0 || a->ld_tables < a->max_blocks || a->layers < 0 || a->num_pages < 0) return refuse(op, "bad sizes");
  if (a->max_path < 1 || a->max_path > 256) return refuse(op, "paths of 1 to 256 rows");
  if (a->max_blocks > INT_MAX / tree::kPage) return refuse(op, "positions pass 32 bits");
  if (a->layers && (!a->kv || a->kv_heads < 1 || a->kv_heads > 4096 || a->layer_stride % 8 || a->layer_stride / 4096 < a->num_pages * (a->layers > 1) * a->kv_heads))
    return refuse(op, "layers of the cache are missing, overlap or lie a number of elements apart that 8 does not divide");
  if (a->layers && !aligned(a->kv, 16)) return refuse(op, "the cache is 16-byte aligned");
  if (!a->S) return 0;
  if (!a->starts || !a->ctx || !a->accepted || !a->path || !a->tokens || !a->new_ctx || (a->T && (!a->ids || !a->drafts)) || (a->max_blocks && !a->block_tables)) return refuse(op, "a buffer is missing");
  if (a->new_ctx == a->ctx) return refuse(op, "new_ctx is a buffer of its own");
  if (int rc = require_device()) return rc;
  return launched(op, tree_accept(*a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
