"""Sampling operators: from a step's logits to the tokens that follow, with or without drafts.
Buffers belong to the caller; they are on the device, and so is what they decide.

token_probs(logits, temperature, workspace, probs)
    FP32 probs [T,V] = softmax(logits / temperature) of each row. BF16 or FP32 logits [T,V], FP32
    temperature [T] (None: 1); 0 gives 1 at the first of the largest logits. Rows may lie further
    apart than V; probs may be FP32 logits themselves. Rows of -inf alone give zeros.
verify_drafts(target_probs, draft_probs, tokens, parents, q_starts, uniforms, workspace, path,
              accepted, next_tokens)
    Rows q_starts[s] .. q_starts[s+1]-1 (INT32 [S+1]) of sequence s are its last certain token and
    then drafted ones, at most 63 of them; INT64 tokens [T]; INT32 parents [T] name each row's parent,
    a row before it, by its number in the sequence (None: the row before). FP32 target_probs and
    draft_probs [T,V]: in each row what follows its token, by the target and by the drafter. With
    draft_probs, a row's children were drawn from its row there, independently (with replacement);
    without (None), they are certain choices, such as a drafter's best. FP32 uniforms [T] in [0, 1), one a row.
    From row 0 on the children of the last accepted row are tried in order, and one stands by
    rejection sampling with its row's number; where none does, the next token is drawn from what the
    rejections leave of the target's row with the number of row 0. So the tokens are distributed as if
    drawn from the target, whatever the drafter; a sequence of one row is a plain draw.
    INT32 path [T]: a sequence's accepted rows by their numbers (row 0 first), then -1; INT32 accepted
    [S] their count; INT64 next_tokens [S] (-1 without rows or where a row has no weights).

workspace: FP32 [262144], of any content, used by one stream at a time.
"""

import torch

from . import _C  # noqa: F401  (registers torch.ops.consumer_int8.*; fails loudly if unbuilt)

token_probs = torch.ops.consumer_int8.token_probs
verify_drafts = torch.ops.consumer_int8.verify_drafts


@torch.library.register_fake("consumer_int8::token_probs")
def _token_probs_fake(logits, temperature, workspace, probs):
    return None


@torch.library.register_fake("consumer_int8::verify_drafts")
def _verify_drafts_fake(target_probs, draft_probs, tokens, parents, q_starts, uniforms, workspace,
                        path, accepted, next_tokens):
    return None


def new_workspace(device="cuda"):
    """The operators' workspace; one for each stream that calls them."""
    return torch.empty(1 << 18, dtype=torch.float32, device=device)
