"""The state of streaming window attention: ring caches of keys and values that hold the first ``sinks`` tokens and the last
``window`` ones of every sequence (the attention of ``functional.window_attention(..., causal=True)``, token by token).

The reference has no counterpart: its models see whole images."""
import torch

from . import functional as VF


class WindowCache:
    """Caches for ``batch`` sequences of ``heads`` key heads of ``dh``: [batch, heads, slots, dh] each, whatever the sequences'
    length.  ``window`` < 0: no window, ``slots`` tokens at most.  ``lengths`` (int32 [batch], on the GPU) are the tokens seen;
    set an entry to a negative number to leave that sequence out of the steps.

    prefill(q, k, v, lengths)   whole prompts into empty caches; their attention's output
    step(q, k, v)               one token more of every sequence; its attention's output
    """

    def __init__(self, batch, heads, dh, window, sinks=0, slots=None, dtype=torch.bfloat16, device='cuda'):
        if slots is None:
            if window < 0:
                raise ValueError('WindowCache: without a window the number of slots must be given')
            slots = sinks + window + 1
        if sinks < 0 or slots < 1 or window >= 0 and slots < sinks + window + 1:
            raise ValueError(f'WindowCache: {slots} slots cannot hold {sinks} sinks, a window of {window} and the new token')
        self.window, self.sinks = int(window), int(sinks) if window >= 0 else 0
        self.k = torch.zeros(batch, heads, slots, dh, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)

    def reset(self):
        self.lengths.zero_()

    @torch.no_grad()
    def prefill(self, q, k, v, lengths=None, scale=None):
        """q [B, N, Hq, dh], k and v [B, N, heads, dh] of prompts of N (or ``lengths``: int32 [B]) tokens."""
        if self.window < 0 and k.shape[1] > self.k.shape[2]:
            raise ValueError(f'WindowCache: prompts of {k.shape[1]} tokens for {self.k.shape[2]} slots')
        out = VF.window_attention(q, k, v, self.window, sinks=self.sinks, causal=True, scale=scale, lengths=lengths)
        VF.window_cache_fill(k, v, self.k, self.v, sinks=self.sinks, lengths=lengths)
        if lengths is None:
            self.lengths.fill_(k.shape[1])
        else:
            self.lengths.copy_(lengths.clamp(max=k.shape[1]))
        return out

    @torch.no_grad()
    def step(self, q, k, v, scale=None):
        """q [B, Hq, dh], k and v [B, heads, dh] of the next token of every sequence."""
        out = VF.window_decode(q, k, v, self.k, self.v, self.lengths, self.window, sinks=self.sinks, scale=scale)
        self.lengths.add_((self.lengths >= 0).to(torch.int32))
        return out
