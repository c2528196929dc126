"""micro-engram's Engram lookup path on MI355X (gfx950): hand-written HIP kernels behind the
reference's MicroEngram module surface.

    from micro_engram_fork_amd import MicroEngram
    eng = MicroEngram(model_dim=5376, engram_dim=64, num_heads=8, orders=(2, 3, 4), ...).cuda()
    with torch.inference_mode():
        out = eng(hidden, input_ids, position_ids)

Losses over a decoder's logits, for training an engram past next-token text, are in `losses`
(token_logps, distill_loss, preference_loss, policy_loss); head_cross_entropy and head_token_logps there take hidden
states and head in place of logits. `optim` has the optimizers of tables (LazyAdamW) and dense weights (DenseAdamW).

The compute lives in libmicro_engram_amd.so (C-ABI: include/micro_engram.h), built in-tree by
`python -m micro_engram_fork_amd._build`.
"""
from .losses import (distill_loss, head_cross_entropy, head_token_logps, policy_loss, preference_loss,  # noqa: F401
                     token_logps)
from .module import (MicroEngram, attach_engram, check_loaded, default_seed,  # noqa: F401
                     engram_from_spec, find_text_layers, layer_device_dtype, resolve_order_sizes)

__all__ = ["MicroEngram", "attach_engram", "check_loaded", "default_seed", "distill_loss", "engram_from_spec",
           "find_text_layers", "head_cross_entropy", "head_token_logps", "layer_device_dtype", "policy_loss",
           "preference_loss", "resolve_order_sizes", "token_logps"]
