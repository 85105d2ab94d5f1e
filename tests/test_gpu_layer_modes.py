"""The operators of ordinary attention layers inside a model that runs under a dispatch mode: FLOP counting and selective activation
checkpointing work and change no result; modes that record or fake operators are refused."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
from torch.utils.flop_counter import FlopCounterMode

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def _layer(x, w, f):
    """A decoder's attention layer: two heads of queries over one of keys."""
    q, k, v = (x @ w).view(2, 70, 4, 64).split((2, 1, 1), 2)
    q, k = sa.rotary_embedding(q, k, f)
    return sa.causal_attention(q, k, v).flatten(2) @ w[:128, :128]


def _leaves(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    return [(torch.randn(*s, generator=g) * 0.1).to(dtype).to(DEV).requires_grad_(True) for s in ((2, 70, 128), (128, 256))]


def _run(f, context=None):
    x, w = _leaves()
    out = checkpoint(_layer, x, w, f, use_reentrant=False, **({"context_fn": context} if context else {})) if context is not False else _layer(x, w, f)
    return (out.detach(), *torch.autograd.grad(out.float().square().sum(), (x, w)))


def test_checkpoints_and_counters():
    f = sa.rotary_frequencies(64, device=DEV)
    want = _run(f, False)

    def policy(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if "mm" in str(op) else CheckpointPolicy.PREFER_RECOMPUTE

    everything = lambda ctx, op, *args, **kwargs: CheckpointPolicy.MUST_SAVE
    for context in (None, lambda: create_selective_checkpoint_contexts(policy), lambda: create_selective_checkpoint_contexts(everything)):
        for a, b in zip(_run(f, context), want):
            assert torch.equal(a, b)
    with FlopCounterMode(display=False) as counter:
        got = _run(f, False)
    assert counter.get_total_flops() > 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_nothing_of_a_call_is_seen():
    x, w = (t.detach() for t in _leaves())
    q, k, v = (x @ w).view(2, 70, 4, 64).split((2, 1, 1), 2)
    kc, vc = (torch.zeros(2, 80, 1, 64, dtype=x.dtype, device=DEV) for _ in range(2))
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    f = sa.rotary_frequencies(64, device=DEV)
    one = lambda t: t[:, :1].contiguous()
    with _Names() as names:
        sa.cache_append(k, v, kc, vc, lengths)
        sa.causal_attention(q, k, v)
        sa.rotary_embedding(q, k, f)
        sa.causal_attention_forward(q, k, v)
    assert names.seen == []
    lengths.fill_(70)
    want = sa.tree_attention(one(q), one(k), one(v), None, kc, vc, lengths)
    with _Names():
        assert torch.equal(sa.tree_attention(one(q), one(k), one(v), None, kc, vc, lengths), want)


def test_modes_that_record_or_fake_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    q = torch.randn(1, 8, 2, 64, device=DEV)
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(lambda t: sa.causal_attention(t, t, t))(q)
    with FakeTensorMode(), pytest.raises(RuntimeError, match="fake tensors"):
        sa.causal_attention(q, q, q)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises(RuntimeError, match="plain tensors"):
        sa.causal_attention(*[mode.from_tensor(q)] * 3)
