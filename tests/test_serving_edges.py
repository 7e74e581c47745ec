"""Calls of the serving operators that the documentation allows at the edge of what it says, each against the statement in 64 bits or against the
ordinary call."""

import pytest
import torch

from test_paged_and_sampling import BF, _small, build, check_attention, gen, torch_calls  # noqa: F401


# ------------------------------------------------------------------ max_q
def _as_the_library(fake, monkeypatch):
    """The library launches nothing where it is told that there are no tokens; the stand-in computes whatever it is told."""
    from cuda_runtime import native

    compute = fake.b200_attn_paged

    def call(args, stream):
        address = args if isinstance(args, int) else args.value
        return 0 if native.AttnPagedArgs.from_address(address).max_q == 0 else compute(args, stream)

    monkeypatch.setattr(fake, "b200_attn_paged", call, raising=False)


def test_attention_with_too_small_a_bound_on_the_tokens_is_computed(fake_native, monkeypatch):
    from paged_attention import paged_attention

    _as_the_library(fake_native, monkeypatch)
    a = {**_small(), "q": gen((3, 4, 64), seed=1), "k_pages": gen((4, 2, 16, 64), seed=2), "v_pages": gen((4, 2, 16, 64), seed=3)}
    want = paged_attention(**a)
    for max_q in (0, 1, 2):
        out = torch.full_like(want, 7.0)
        assert torch.equal(paged_attention(**{**a, "max_q": max_q}, out=out), want)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 70)], [(40, 300), (0, 9), (1, 70)], [(0, 5), (0, 0)]])
def test_attention_whose_bound_on_the_tokens_is_none(native_lib, seqs):
    """max_q = 0 with tokens there: as every other bound that is too small.  Without tokens nothing is written."""
    from paged_attention import paged_attention

    a, start, table = build(seqs, seed=21, extra_tokens=2)
    out = torch.full((start[-1] + 2, 12, 128), 7.0, dtype=BF, device="cuda")
    got = paged_attention(**{**a, "max_q": 0}, out=out)
    check_attention(got, a, start, table, seqs)
    assert (got[start[-1]:] == 7).all()
