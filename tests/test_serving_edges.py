"""Calls of the serving operators that the documentation allows at the edge of what it says, each against the statement in 64 bits or against the
ordinary call."""

import random

import numpy as np
import pytest
import torch

from test_paged_and_sampling import BF, _small, build, check_attention, check_draw, gen, torch_calls  # noqa: F401


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


# ------------------------------------------------------------------ Sampler
def _held(x):
    """Elements of the tensors in an object's attributes, views counted as if they were not."""
    if isinstance(x, torch.Tensor):
        return x.numel()
    if isinstance(x, dict):
        return sum(_held(v) for v in x.values())
    return sum(_held(v) for v in x) if isinstance(x, (tuple, list)) else _held(vars(x)) if hasattr(x, "settings") else 0


def test_sampler_does_not_keep_a_set_of_settings_for_every_batch_size(fake_native):
    """A server's batch grows and shrinks: what a sampler holds is bounded by the largest, and every batch draws as a sampler of its own would."""
    from sampling import Sampler

    sizes = [*range(1, 65), *range(64, 0, -1), 7, 200, 7]
    logits = gen((200, 30), torch.float32, 1)
    sampler = Sampler(temperature=0.9, top_k=7, top_p=0.8, min_p=0.01, seed=3)
    g = torch.Generator().manual_seed(3)
    from sampling import sample_rows

    for rows in sizes:
        u = torch.rand(rows, generator=g)
        full = lambda v, dt=torch.float32: torch.full((rows,), v, dtype=dt)
        want = sample_rows(logits[:rows], u, full(0.9), full(7, torch.int32), full(0.8), full(0.01))
        assert torch.equal(sampler(logits[:rows]), want)
    # four settings of one number, for the powers of two up to 256, and views of the last batch
    assert _held(sampler) <= 4 * (1 + 511 + 200)


def test_sampler_of_one_setting_per_row_takes_batches_of_that_size_alone(fake_native):
    from sampling import Sampler

    sampler = Sampler(temperature=[0.5, 1.0, 0.0])
    logits = gen((4, 30), torch.float32, 2)
    assert sampler(logits[:3])[2] == logits[2].argmax()
    for rows in (1, 2, 4):
        with pytest.raises(ValueError, match="one for each"):
            sampler(logits[:rows])
    assert sampler(logits[:3])[2] == logits[2].argmax()
    assert Sampler(temperature=[0.0])(logits[:1])[0] == logits[0].argmax()
    assert Sampler()(logits[:0]).shape == (0,)


# ------------------------------------------------------------------ QwenSession
def _session(T=8, S=16, B=2):
    import model_zoo as mz
    from ir_export import extract_ir
    from qwen_session import QwenSession
    from test_checkpoint_session import _tiny

    cfg, sd, model = _tiny()
    L = cfg.num_hidden_layers
    irp = extract_ir(mz.QwenPrefillWrapper(model), mz.qwen2_example_inputs(cfg, B, T, None, device="cpu"), "p")
    ird = extract_ir(mz.QwenDecodeWrapper(model, L), mz.qwen2_example_inputs(cfg, B, 1, S, device="cpu"), "d")
    ids = torch.randint(0, cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(4)).numpy()
    return QwenSession(irp, ird, mz.state_dict_numpy(sd), L), ids


def test_session_does_not_draw_from_a_row_that_the_prompt_does_not_have(fake_native):
    """A prompt of no tokens has no last row: counted from the end, it would be that of the padding."""
    from sampling import Sampler

    T = 8
    sess, ids = _session(T)
    for n in (1, T):
        assert (sess.prefill(ids, n, sampler=Sampler(temperature=0.0)) == sess.prefill(ids, n)).all()
    for n in (0, -1, -T, T + 1):
        sess.position = 5
        with pytest.raises(ValueError, match="prompt"):
            sess.prefill(ids, n, sampler=Sampler())
        assert sess.position == 5


def test_session_takes_a_step_again_whose_token_could_not_be_drawn(fake_native):
    from sampling import Sampler

    sess, ids = _session()
    first, steps = sess.prefill(ids), []
    for _ in range(3):
        steps.append((sess.step(first), sess.position, sess.last_logits.to_numpy().copy()))
    sess.prefill(ids)
    for tok, position, logits in steps:
        with pytest.raises(ValueError, match="one for each"):
            sess.step(first, sampler=Sampler(top_k=[1, 2, 3]))
        assert (sess.step(first) == tok).all() and sess.position == position
        assert (sess.last_logits.to_numpy() == logits).all()


# ------------------------------------------------------------------ attention: many sequences, starts out of range
def _many(n, tokens, keys, seed):
    """`n` sequences: one token each but for a few of up to `tokens`, 1 to `keys` keys, some without any."""
    r = random.Random(seed)
    seqs = []
    for i in range(n):
        T = r.randint(2, tokens) if tokens > 1 and i % 9 == 4 else 1
        seqs.append((0, r.randint(0, keys)) if i % 31 == 7 else (T, 0) if i % 97 == 50 else (T, max(T, r.randint(1, keys))))
    return seqs


# How the work is dealt out: up to 32 sequences (one warp), more (all threads), more than a block has threads (256 or 352; several of each), more
# pieces in a block than a list holds (32: the block goes on with a second list over the same rings), items whole (narrow tables) and cut (wide ones).
MANY = {
    "chunks_33": dict(seqs=_many(33, 60, 900, 1)),
    "chunks_60_wide": dict(seqs=_many(60, 60, 900, 2), table_extra=40),
    "chunks_400_fp16_d64": dict(seqs=_many(400, 70, 600, 3), heads=(14, 2), dim=64, dtype=torch.float16, page=48),
    "chunks_400_window": dict(seqs=_many(400, 40, 700, 4), window=100, table_extra=40),
    "decode_300_wide": dict(seqs=_many(300, 1, 400, 5), table_extra=60),
    "decode_600_8_heads": dict(seqs=_many(600, 1, 300, 6), heads=(16, 8), dim=64),
    "draft_600_8_heads_wide": dict(seqs=_many(600, 4, 300, 7), heads=(16, 8), dim=64, dtype=torch.float16, table_extra=130),
    "decode_4096": dict(seqs=_many(4096, 1, 100, 8)),
    "decode_4096_wide_window": dict(seqs=_many(4096, 1, 100, 9), table_extra=70, window=33),
    "chunks_4096": dict(seqs=_many(4096, 25, 100, 10), heads=(6, 2)),
    "chunks_4096_wide": dict(seqs=_many(4096, 25, 100, 11), heads=(6, 2), table_extra=40),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", MANY)
def test_attention_of_many_sequences(native_lib, name):
    from paged_attention import paged_attention

    case = MANY[name]
    a, start, table = build(**case, seed=len(name), extra_tokens=3)
    N = a["q"].shape[0]
    room = torch.full((N + 8, *a["q"].shape[1:]), 7.0, dtype=a["q"].dtype, device="cuda")
    out = room[4:4 + N]
    paged_attention(**a, window=case.get("window", 0), out=out)
    torch.cuda.synchronize()
    check_attention(out, a, start, table, case["seqs"], case.get("window", 0))
    assert (room[:4] == 7).all() and (room[4 + start[-1]:] == 7).all()
    first = out.clone()
    paged_attention(**a, window=case.get("window", 0), out=out)
    assert torch.equal(out, first)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 70)], [(40, 300), (1, 70)], [(1, 5000), (2, 4000)]])
def test_attention_cuts_starts_to_the_tokens_that_are_there(native_lib, seqs):
    """A first token ahead of the first and a last one behind the last: results are those of the tokens in between, nothing is written beside them."""
    from paged_attention import paged_attention

    a, start, table = build(seqs, seed=3, extra_tokens=5)
    N = a["q"].shape[0]
    room = torch.full((N + 16, 12, 128), 7.0, dtype=BF, device="cuda")
    a["q_start"][0], a["q_start"][2] = -4, 1 << 30
    paged_attention(**a, out=room[8:8 + N])
    cut = [0, start[1], N]
    check_attention(room[8:8 + N], a, cut, table, [(start[1], seqs[0][1]), (N - start[1], seqs[1][1])])
    assert (room[:8] == 7).all() and (room[8 + N:] == 7).all()


# ------------------------------------------------------------------ the draw
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_draw_from_the_longest_flat_row(native_lib, dtype):
    """4194304 equal tokens of weight 2^40 each: their sum is 2^62, and all of it is exact."""
    x = torch.full((3, 1 << 22), -2.5, dtype=dtype)
    u = np.array([0.0, 0.6180339, 1.0 - 2.0 ** -24])
    check_draw(x, u)
    check_draw(x, u, top_k=np.full(3, 3000001))
    check_draw(x, u, top_p=np.full(3, 0.75), min_p=np.ones(3))
