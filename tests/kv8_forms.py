"""The forms that the 8-bit pool's attention takes, each by the arguments that choose it."""
from __future__ import annotations

import torch

from kv8_helpers import dev, host

FAR = 20000  # a bound on the lengths behind which contexts are cut


def attend(form, pool, b, q, dtype, scale=None, zero_sink=False):
    """Attention of batch b's new rows q: "seq" and "split" decode, "whole" and "cut" extend.
    Without room for partials there are no pieces; long bounds make some."""
    kw = dict(scale=scale, zero_sink=zero_sink)
    if form in ("seq", "whole"):
        kw.update(workspace=torch.empty(0, dtype=torch.uint8, device="cuda"), max_ctx_len=max(b.ctx))
    else:
        kw.update(max_ctx_len=max(FAR, *b.ctx))
    if form in ("seq", "split"):
        o = pool.decode_attention(0, dev(q, dtype), *b.device(), **kw)
    else:
        o = pool.extend_attention(0, dev(q, dtype), b.q_indptr(), *b.device(), max_q_len=max(b.new), **kw)
    pool.check()
    return host(o)


def chunks(form, ctx, most):
    """New tokens per sequence: one in decode, up to `most` in extend."""
    return [1] * len(ctx) if form in ("seq", "split") else [min(c, most) for c in ctx]
