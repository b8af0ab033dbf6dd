"""The plain models with keys and values held in 4 bits, and tokens whose keys and values lie off the borders between codes
(an engine in 32-bit rounds them differently by some 1e-6, and a code that turns is a whole step)."""

import contextlib

import torch

import plain_gpt2
import plain_int4


@contextlib.contextmanager
def cache_in_4_bits(margins=None):
    """While active, ``plain_gpt2`` attends over what a cache in 4 bits holds.  ``margins`` (a list) collects how near any
    element comes to a border, in steps."""
    attend = plain_gpt2.causal_attention

    def over_codes(q, k, v, scale, window=0):
        held = []
        for x in (k, v):
            rows = x.transpose(0, 1).reshape(x.shape[1], -1)
            codes, steps, values = plain_int4.held(rows.float(), x.shape[0])
            if margins is not None:
                per = torch.from_numpy(steps).repeat_interleave(32, dim=2)[..., :x.shape[2]]
                ratio = x.transpose(0, 1) / per
                # (beyond the outermost codes there is no border)
                near = ((ratio - 0.5) - (ratio - 0.5).round()).abs()
                margins.append(float(near[(ratio > -8.4) & (ratio < 7.4)].min()))
            held.append(values.view(x.shape[1], x.shape[0], -1).transpose(0, 1))
        return attend(q, *held, scale, window)

    plain_gpt2.causal_attention = over_codes
    try:
        yield
    finally:
        plain_gpt2.causal_attention = attend
