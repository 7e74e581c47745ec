"""Append to a paged cache, attention over its pages, drawing tokens: host logic and refusals here (CPU), kernels in the gpu tests,
each against a statement in 64 bits."""

import ctypes as C
import itertools
import random

import numpy as np
import pytest
import torch

import serving_reference as ref

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def torch_calls():
    import build_native

    build_native.build_torch_calls()


def gen(shape, dtype=BF, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


# ------------------------------------------------------------------ host logic
def test_pages_are_handed_out_as_sequences_grow_and_come_back(fake_native):
    from paged_attention import PagedKVCache

    cache = PagedKVCache(6, 16, 1, 2)
    a, b = cache.open(), cache.open()
    st = cache.step([a, b], [17, 3])
    assert cache.free_pages == 3 and st.max_q == 17 and st.n_tokens == 20
    assert st.q_start.tolist() == [0, 17, 20] and st.kv_len.tolist() == [17, 3] and st.last.tolist() == [16, 19]
    assert st.positions.tolist() == [*range(17), 0, 1, 2]
    assert len(set(st.slots.tolist())) == 20
    st = cache.step([b, a], [1, 15])
    assert cache.free_pages == 3 and st.kv_len.tolist() == [4, 32] and st.positions.tolist() == [3, *range(17, 32)]
    before = (cache.length(a), cache.length(b), cache.free_pages)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.step([a, b], [48, 16])
    assert before == (cache.length(a), cache.length(b), cache.free_pages)
    cache.close(a)
    assert cache.free_pages == 5
    with pytest.raises(ValueError, match="no such sequence"):
        cache.step([a], [1])
    for seqs, new in (([b, b], [1, 1]), ([b], [0]), ([], []), ([b], [1, 2])):
        with pytest.raises(ValueError):
            cache.step(seqs, new)
    for kw in ({"page_size": 8}, {"page_size": 24}, {"head_dim": 96}, {"dtype": F32}, {"num_pages": 0}):
        with pytest.raises(ValueError):
            PagedKVCache(**{"num_pages": 2, "page_size": 16, "num_layers": 1, "num_kv_heads": 1, **kw})


def _small():
    kp = torch.zeros(4, 2, 16, 64, dtype=BF)
    return {"q": torch.zeros(3, 4, 64, dtype=BF), "k_pages": kp, "v_pages": kp.clone(), "q_start": torch.tensor([0, 3], dtype=torch.int32),
            "kv_len": torch.tensor([3], dtype=torch.int32), "page_table": torch.zeros(1, 2, dtype=torch.int32), "max_q": 3}


@pytest.mark.parametrize("change", [
    {"q": torch.zeros(3, 4, 64)}, {"q": torch.zeros(3, 256, dtype=BF)}, {"k_pages": torch.zeros(8, 16, 64, dtype=BF)}, {"kv_len": torch.zeros((), dtype=torch.int32)}, {"q": torch.zeros(3, 4, 128, dtype=BF)}, {"q": torch.zeros(3, 64, 4, dtype=BF).transpose(1, 2)},
    {"v_pages": torch.zeros(4, 2, 32, 64, dtype=BF)}, {"q_start": torch.tensor([0, 3])}, {"q_start": torch.tensor([0, 1, 3], dtype=torch.int32)},
    {"kv_len": torch.tensor([3])}, {"page_table": torch.zeros(2, 2, dtype=torch.int32)}, {"page_table": torch.zeros(1, 2)},
    {"out": torch.zeros(3, 4, 64)}, {"out": torch.zeros(2, 4, 64, dtype=BF)}])
def test_attention_refuses_on_the_host(fake_native, change):
    from paged_attention import paged_attention

    with pytest.raises(ValueError):
        paged_attention(**{**_small(), **change})
    assert "attn_paged" not in fake_native.calls


@pytest.mark.parametrize("change", [
    {"v": torch.zeros(3, 1, 64, dtype=BF)}, {"k": torch.zeros(3, 2, 64, dtype=HF)}, {"slots": torch.zeros(3, dtype=torch.int32)},
    {"slots": torch.zeros(2, dtype=torch.int64)}, {"cos": None}, {"cos": torch.zeros(3, 32)}, {"q": torch.zeros(2, 4, 64, dtype=BF)},
    {"q_out": torch.zeros(3, 4, 128, dtype=BF)}, {"sin": torch.zeros(3, 64, dtype=BF)}])
def test_append_refuses_on_the_host(fake_native, change):
    from paged_attention import paged_append

    kp = torch.zeros(4, 2, 16, 64, dtype=BF)
    args = {"q": torch.zeros(3, 4, 64, dtype=BF), "k": torch.zeros(3, 2, 64, dtype=BF), "v": torch.zeros(3, 2, 64, dtype=BF), "cos": torch.zeros(3, 64),
            "sin": torch.zeros(3, 64), "k_pages": kp, "v_pages": kp.clone(), "slots": torch.zeros(3, dtype=torch.int64)}
    with pytest.raises(ValueError):
        paged_append(**{**args, **change})
    assert "paged_append" not in fake_native.calls


@pytest.mark.parametrize("change", [
    {"logits": torch.zeros(2, 8, dtype=torch.int32)}, {"logits": torch.zeros(8, 2).t()}, {"logits": torch.zeros(2, 0)}, {"uniform": None},
    {"uniform": torch.zeros(2, dtype=torch.float64)}, {"uniform": torch.zeros(3)}, {"top_k": torch.zeros(2)}, {"temperature": torch.ones(1)},
    {"top_p": torch.ones(2, 1)}, {"min_p": torch.ones(2, dtype=HF)}, {"out": torch.zeros(2, dtype=torch.int32)}])
def test_sampling_refuses_on_the_host(fake_native, change):
    from sampling import sample_rows

    with pytest.raises(ValueError):
        sample_rows(**{"logits": torch.zeros(2, 8), "uniform": torch.zeros(2), **change})
    assert "sample_rows" not in fake_native.calls


def _attn_args(**change):
    """Arguments of b200_attn_paged with made-up addresses: a call that must be refused before anything is launched."""
    from cuda_runtime import native

    a = dict(q=4096, k_pages=4096, v_pages=4096, out=4096, q_start=4096, kv_len=4096, page_table=4096, workspace=4096, workspace_bytes=1 << 30, B=1, n_tokens=3,
             max_q=3, num_pages=4, table_stride=2, q_strides=(256, 64), kv_strides=(2048, 1024, 64), window=0, Hq=4, Hkv=2, D=64, page_size=16, dtype=2, scale=0.125)
    assert set(change) <= set(a)
    return C.byref(native.AttnPagedArgs(**{**a, **change}))


@pytest.mark.parametrize("change,code", [
    ({"q": 0}, -1), ({"page_table": 0}, -1), ({"D": 96}, -1), ({"Hq": 5}, -1), ({"Hq": 512, "Hkv": 2}, -1), ({"page_size": 24}, -1), ({"page_size": 0}, -1),
    ({"window": -1}, -1), ({"B": -1}, -1), ({"table_stride": 0}, -1), ({"workspace": 0}, -1), ({"workspace_bytes": 100}, -1), ({"q": 4098}, -2), ({"out": 4104}, -2),
    ({"workspace": 4104}, -2), ({"q_strides": (256, 60)}, -2), ({"q_strides": (256, 0)}, -2), ({"kv_strides": (2048, 1024, -64)}, -2),
    ({"kv_strides": (0, 1024, 64)}, -2), ({"dtype": 0}, -4), ({"table_stride": 1 << 28}, -5), ({"B": 4097}, -5)])
def test_library_refuses_attention_calls(native_lib, change, code):
    assert native_lib.b200_attn_paged(_attn_args(**change), 0) == code
    assert native_lib.b200_last_error()


@pytest.mark.parametrize("change,code", [({"k": 0}, -1), ({"q_out": 0}, -1), ({"cos_t": 0}, -1), ({"D": 24}, -1), ({"page_size": 0}, -1), ({"k": 4104}, -2),
                                         ({"v_strides": (128, 4)}, -2), ({"table_dtype": 1}, -4), ({"dtype": 0}, -4)])
def test_library_refuses_append_calls(native_lib, change, code):
    from cuda_runtime import native

    a = dict(q=4096, k=4096, v=4096, cos_t=4096, sin_t=4096, q_out=4096, k_pages=4096, v_pages=4096, slots=4096, n_tokens=3, num_pages=4, q_strides=(256, 64),
             k_strides=(128, 64), v_strides=(128, 64), kv_strides=(2048, 1024, 64), Hq=4, Hkv=2, D=64, page_size=16, table_dtype=0, dtype=2)
    assert native_lib.b200_paged_append(C.byref(native.PagedAppendArgs(**{**a, **change})), 0) == code


@pytest.mark.parametrize("change,code", [({"logits": 0}, -1), ({"uniform": 0}, -1), ({"cols": 0}, -1), ({"cols": (1 << 22) + 1}, -5), ({"rows": 65536}, -5),
                                         ({"dtype": 3}, -4)])
def test_library_refuses_sampling_calls(native_lib, change, code):
    a = dict(logits=4096, out=4096, rows=2, cols=8, row_stride=8, temperature=0, top_k=0, top_p=0, min_p=0, uniform=4096, dtype=0, stream=0)
    a.update(change)
    assert native_lib.b200_sample_rows(*a.values()) == code


def test_library_refuses_to_append_to_expanded_pages(native_lib):
    """Rows of all heads (or pages) in one place would be written at once."""
    from cuda_runtime import native

    a = dict(q=4096, k=4096, v=4096, cos_t=4096, sin_t=4096, q_out=4096, k_pages=4096, v_pages=4096, slots=4096, n_tokens=3, num_pages=4, q_strides=(256, 64),
             k_strides=(128, 64), v_strides=(128, 64), Hq=4, Hkv=2, D=64, page_size=16, table_dtype=0, dtype=2)
    for strides in ((0, 1024, 64), (2048, 0, 64), (2048, 1024, 0), (2048, 1024, -64)):
        assert native_lib.b200_paged_append(C.byref(native.PagedAppendArgs(**a, kv_strides=strides)), 0) == -2


def test_tensors_in_host_memory_do_not_reach_the_library(native_lib):
    from paged_attention import paged_append, paged_attention
    from sampling import sample_rows

    kp = torch.zeros(4, 2, 16, 64, dtype=BF)
    for call in (lambda: paged_attention(**_small()), lambda: sample_rows(torch.zeros(2, 8), torch.zeros(2)),
                 lambda: paged_append(None, torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF), None, None, kp, kp.clone(), torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_sampler_keeps_the_settings_it_was_made_with(fake_native):
    from sampling import Sampler

    temperature = torch.zeros(2)
    logits = torch.randn(2, 50, generator=torch.Generator().manual_seed(1))
    sampler, greedy = Sampler(temperature=temperature), logits.argmax(1)
    temperature += 5.0
    assert torch.equal(sampler(logits), greedy)
    temperature += 5.0
    assert torch.equal(sampler(logits), greedy)


def test_empty_calls_launch_nothing(native_lib):
    for change in ({"B": 0}, {"n_tokens": 0}, {"max_q": 0}):
        assert native_lib.b200_attn_paged(_attn_args(**change), 0) == 0
    assert native_lib.b200_sample_rows(4096, 4096, 0, 8, 8, None, None, None, None, 4096, 0, 0) == 0


def test_session_draws_tokens(fake_native):
    """`generate` with a sampler: the tokens are those that `sample_rows` gives for the session's own logits and the generator's numbers; temperature 0
    is the greedy session."""
    import model_zoo as mz
    from ir_export import extract_ir
    from qwen_session import QwenSession
    from sampling import Sampler
    from test_checkpoint_session import _tiny

    cfg, sd, model = _tiny()
    L, T, S, B = cfg.num_hidden_layers, 16, 40, 2
    irp = extract_ir(mz.QwenPrefillWrapper(model), mz.qwen2_example_inputs(cfg, B, T, None, device="cpu"), "p")
    ird = extract_ir(mz.QwenDecodeWrapper(model, L), mz.qwen2_example_inputs(cfg, B, 1, S, device="cpu"), "d")
    sess = QwenSession(irp, ird, mz.state_dict_numpy(sd), L)
    ids = torch.randint(0, cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(4)).numpy()
    greedy = sess.generate(ids, 4, prompt_len=11)
    np.testing.assert_array_equal(sess.generate(ids, 4, prompt_len=11, sampler=Sampler(temperature=0.0)), greedy)
    seen = []

    class Watched(Sampler):
        def __call__(self, logits):
            seen.append((logits.clone(), super().__call__(logits)))
            return seen[-1][1]

    got = sess.generate(ids, 4, prompt_len=11, sampler=Watched(temperature=[0.8, 1.2], top_k=50, top_p=0.9, seed=3))
    g = torch.Generator().manual_seed(3)
    for i, (logits, tokens) in enumerate(seen):
        u = torch.rand(B, generator=g)
        temp, p = np.float32([0.8, 1.2]), np.float32([0.9, 0.9])
        assert tokens.tolist() == ref.draw(logits.double().numpy(), u.numpy(), temp, [50, 50], p)
        np.testing.assert_array_equal(got[:, i], tokens.numpy())
    with pytest.raises(ValueError, match="one for each"):
        sess.generate(ids, 2, sampler=Sampler(top_k=[1, 2, 3]))


# ------------------------------------------------------------------ attention on the GPU
def build(seqs, heads=(12, 2), dim=128, page=16, dtype=BF, window=0, seed=0, spare=2, poison=True, rows_first=False, extra_tokens=0, table_extra=2):
    """A batch on the GPU.  Every row of the pages that no token may look at is NaN or infinite, and table entries that nobody may look at lie far outside."""
    r = random.Random(seed)
    need = [-(-n // page) for _, n in seqs]
    n_pages = sum(need) + spare
    order = list(range(n_pages))
    r.shuffle(order)
    width = max(need + [0]) + table_extra
    table = [[r.choice((-1, 1 << 30, -(1 << 31)))] * width for _ in seqs]
    Hq, Hkv = heads
    shape = (n_pages, Hkv, page, dim)
    if poison:
        k, v = torch.full(shape, float("nan"), dtype=dtype), torch.full(shape, float("inf"), dtype=dtype)
    else:
        k, v = gen(shape, dtype, seed + 5), gen(shape, dtype, seed + 6)
    for b, (T, n) in enumerate(seqs):
        lo = max(0, n - T - window + 1) if window else 0
        for i in range(need[b]):
            at = order.pop()
            a, z = max(lo, i * page), min(n, (i + 1) * page)
            if a < z:
                table[b][i] = at
                k[at, :, a - i * page:z - i * page] = gen((Hkv, z - a, dim), dtype, seed + 1000 * b + 7 * i + 1)
                v[at, :, a - i * page:z - i * page] = gen((Hkv, z - a, dim), dtype, seed + 1000 * b + 7 * i + 2)
    if rows_first:   # [pages, rows, heads, D] in memory
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    start = [0, *itertools.accumulate(T for T, _ in seqs)]
    N = start[-1] + extra_tokens
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    return {"q": gen((N, Hq, dim), dtype, seed + 3, 1.2).cuda(), "k_pages": k.cuda(), "v_pages": v.cuda(), "q_start": i32(start), "kv_len": i32([n for _, n in seqs]),
            "page_table": i32(table), "max_q": max(T for T, _ in seqs)}, start, table


def check_attention(got, a, start, table, seqs, window=0, scale=None):
    """Per value: the output's own rounding and those of the probabilities, half a step each (eps / 2 of |out| and of sum(p |v|)); what a probability
    loses below the smallest normal number of fp16 (half of 2^-24 each, the largest of a row being at least 1); scores are fp32 sums of up to 128
    products, relative 128 * 2^-24 of sum |q k| scale (below 30 here), so 2.3e-4 of a probability at worst, half of which moves numerator against sum,
    and merging, exponentials and sums another 2^-20: 3e-4 of sum(p |v|)."""
    D, dtype = a["q"].shape[2], a["q"].dtype
    want, spread, flat = ref.attention(a["q"], a["k_pages"], a["v_pages"], start, [n for _, n in seqs], table, D ** -0.5 if scale is None else scale, window)
    half = torch.finfo(dtype).eps / 2
    tol = half * (want.abs() + spread) * 1.01 + 3e-4 * spread + (2 ** -25 * flat + 2 ** -25 if dtype == HF else 0) + 1e-30
    n = start[-1]
    got = got.cpu()
    assert not got[:n].isnan().any()
    bad = ((got[:n].double() - want[:n]).abs() > tol[:n]).nonzero()
    assert len(bad) == 0, (len(bad), bad[:4].tolist(), got[tuple(bad[0])], want[tuple(bad[0])])


CASES = {
    "one_token": dict(seqs=[(1, 1)]),
    "edges": dict(seqs=[(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 613)]),
    "edges_page48": dict(seqs=[(1, n) for n in (1, 47, 48, 49, 95, 96, 97, 144, 145, 500)], page=48),
    "empty_and_short": dict(seqs=[(1, 0), (0, 40), (1, 5), (0, 0), (3, 2), (2, 0), (1, 33)]),
    "all_empty": dict(seqs=[(0, 0), (0, 7), (1, 0)]),
    "decode_long": dict(seqs=[(1, 20001)], page=64),
    "decode_ragged": dict(seqs=[(1, 1 + (i * 977) % 3001) for i in range(40)]),
    "decode_mha": dict(seqs=[(1, 300), (1, 1000), (1, 31)], heads=(6, 6), page=32),
    "decode_16_heads": dict(seqs=[(1, 300), (1, 1111)], heads=(16, 1)),
    "decode_17_heads": dict(seqs=[(1, 300), (1, 1111), (1, 5)], heads=(34, 2)),
    "decode_d64": dict(seqs=[(1, 129), (1, 1000), (1, 64)], heads=(14, 2), dim=64),
    "decode_window": dict(seqs=[(1, n) for n in (5, 99, 100, 101, 116, 117, 900, 901, 2500)], window=100),
    "decode_window_1": dict(seqs=[(1, 1), (1, 16), (1, 17), (1, 300)], window=1),
    "draft_4": dict(seqs=[(4, 300), (4, 4), (3, 700), (1, 50), (4, 129)], heads=(16, 8), dim=64, page=32, dtype=HF),
    "draft_2_window": dict(seqs=[(2, 300), (2, 65), (1, 700), (2, 2)], window=64),
    "chunk": dict(seqs=[(100, 900)]),
    "chunk_long_history": dict(seqs=[(9, 9000)]),   # some seventy pieces to join
    "chunk_long_history_d64": dict(seqs=[(30, 6000), (1, 50), (2, 3000)], heads=(14, 2), dim=64, dtype=HF),
    "chunk_odd": dict(seqs=[(131, 131), (1, 900), (77, 1300), (21, 21), (22, 150), (0, 9), (63, 64)], page=48),
    "chunk_window": dict(seqs=[(131, 531), (1, 900), (300, 300), (50, 2000)], window=77),
    "chunk_window_fp16_d64": dict(seqs=[(257, 600), (1, 900), (40, 41)], window=128, heads=(14, 2), dim=64, dtype=HF, page=256),
    "prompt": dict(seqs=[(700, 700)], page=64),
    "prompt_mha_fp16": dict(seqs=[(300, 300), (129, 400)], heads=(3, 3), dtype=HF, page=32),
    "prompt_mqa": dict(seqs=[(90, 200), (1, 1)], heads=(40, 1)),
    "prompt_100_heads": dict(seqs=[(5, 200), (9, 9)], heads=(100, 1), dim=64),
    "short_of_keys": dict(seqs=[(200, 50), (40, 3), (7, 7)]),
    "page_1008": dict(seqs=[(1, 2000), (150, 1500)], page=1008),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_attention(native_lib, name):
    from paged_attention import paged_attention

    case = CASES[name]
    a, start, table = build(**case, seed=len(name))
    got = paged_attention(**a, window=case.get("window", 0))
    torch.cuda.synchronize()
    check_attention(got, a, start, table, case["seqs"], case.get("window", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 70)], [(40, 300), (1, 70)]])
def test_attention_layouts_rows_behind_and_other_scales(native_lib, seqs):
    from paged_attention import paged_attention

    a, start, table = build(seqs, rows_first=True, extra_tokens=5, seed=2)
    N = a["q"].shape[0]
    wide = torch.zeros(N, 16, 128, dtype=BF, device="cuda")   # the columns of a merged projection
    wide[:, :12] = a["q"]
    a["q"] = wide[:, :12]
    for scale in (None, 0.0, -0.05, 1.0):
        out = torch.full((N, 12, 128), 7.0, dtype=BF, device="cuda")
        paged_attention(**a, scale=scale, out=out)
        check_attention(out, a, start, table, seqs, scale=scale)
        assert (out[start[-1]:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 70)], [(40, 300), (1, 70)]])
def test_attention_reads_pages_that_are_not_there_as_zeros_and_cuts_lengths(native_lib, seqs):
    """Page ids outside the cache, lengths past the table, starts past the tokens: cut to what there is, nothing is read or written outside."""
    from paged_attention import paged_attention

    a, start, table = build(seqs, seed=3, table_extra=0)
    for b, i, bad in ((0, 3, 1 << 29), (0, 7, -5)):
        table[b][i] = bad
    a["page_table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    check_attention(paged_attention(**a), a, start, table, seqs)
    a["kv_len"][0] = 1 << 30          # cut to the table: 19 pages of 16 rows
    a["kv_len"][1] = -7               # no keys: zeros
    out = torch.full_like(a["q"], 7.0)
    full = {**a, "k_pages": torch.nan_to_num(a["k_pages"], 0.0), "v_pages": torch.nan_to_num(a["v_pages"], 0.0, 0.0, 0.0)}
    paged_attention(**full, out=out)
    cut = [(seqs[0][0], 19 * 16), (seqs[1][0], 0)]
    check_attention(out, full, start, table, cut)
    a["q_start"][2] = 1 << 30
    a["q_start"][0] = -4
    paged_attention(**full | {"q_start": a["q_start"]}, out=out)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 300), (3, 1)], [(40, 300), (60, 17)]])
@pytest.mark.parametrize("window", [(1 << 30) - 1, 1 << 30, (1 << 63) - 1])
def test_attention_windows_longer_than_any_sequence(native_lib, seqs, window):
    """As if there were none, for tokens ahead of position 0 too."""
    from paged_attention import paged_attention

    a, start, table = build(seqs, seed=4)
    check_attention(paged_attention(**a, window=window), a, start, table, seqs)
    assert torch.equal(paged_attention(**a, window=window), paged_attention(**a))


@pytest.mark.gpu
@pytest.mark.parametrize("T,keys,table_pages", [(1, 300, 20), (1, 20000, 1250), (40, 300, 20), (40, 9000, 600)])
def test_attention_of_a_query_that_is_no_number_gives_none(native_lib, T, keys, table_pages):
    """Whether or not its keys are shared out and joined again; its neighbours do not notice."""
    from paged_attention import paged_attention

    a, start, table = build([(T, keys)], seed=5, table_extra=table_pages - -(-keys // 16))
    broken = a["q"].clone()
    broken[T // 2, 3] = float("nan")
    got = paged_attention(**{**a, "q": broken})
    assert got[T // 2, 3].isnan().all()
    got[T // 2, 3] = paged_attention(**a)[T // 2, 3]
    check_attention(got, a, start, table, [(T, keys)])


@pytest.mark.gpu
def test_attention_over_a_cache_past_32_bits(native_lib):
    from paged_attention import paged_attention

    pages = torch.empty(150000, 2, 64, 128, dtype=BF, device="cuda")   # 2.46e9 elements
    small = gen((8, 2, 64, 128), seed=1)
    for i, at in enumerate((149999, 131071, 131072, 149000, 0, 140001, 149990, 131073)):
        pages[at] = small[i].cuda()
    for T in (1, 50):
        q, start, table = gen((T, 12, 128), seed=2).cuda(), [0, T], [[149999, 131071, 131072, 149000, 0, 140001, 149990, 131073]]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        got = paged_attention(q, pages, pages, i32(start), i32([500]), i32(table), T)
        host = {"q": q, "k_pages": small, "v_pages": small}
        check_attention(got, host, start, [list(range(8))], [(T, 500)])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,later", [([(1, 300), (1, 70), (1, 2000)], [(1, 900), (1, 0), (1, 17)]),
                                        ([(40, 300), (1, 70), (1, 2000)], [(1, 30), (100, 1700), (0, 50)])])
def test_attention_is_captured_and_follows_its_index_tensors(native_lib, seqs, later):
    """A captured call replayed after lengths, starts, pages and queries have changed; two captured graphs on two streams at once."""
    from paged_attention import paged_attention

    a, start, table = build(later, seed=4, spare=1)
    b, start_b, table_b = build(seqs, seed=5, spare=1)
    width, N = max(a["page_table"].shape[1], b["page_table"].shape[1]), max(a["q"].shape[0], b["q"].shape[0])
    pages = max(a["k_pages"].shape[0], b["k_pages"].shape[0])
    live = {"q": torch.zeros(N, 12, 128, dtype=BF, device="cuda"), "k_pages": torch.zeros(pages, 2, 16, 128, dtype=BF, device="cuda"),
            "v_pages": torch.zeros(pages, 2, 16, 128, dtype=BF, device="cuda"), "q_start": torch.zeros(4, dtype=torch.int32, device="cuda"),
            "kv_len": torch.zeros(3, dtype=torch.int32, device="cuda"), "page_table": torch.full((3, width), -1, dtype=torch.int32, device="cuda"),
            "max_q": max(a["max_q"], b["max_q"])}

    def put(src):
        for key in ("q", "k_pages", "v_pages", "q_start", "kv_len"):
            live[key][:src[key].shape[0]] = src[key]
        live["page_table"][:, :src["page_table"].shape[1]] = src["page_table"]

    put(b)
    paged_attention(**live)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(paged_attention(**live))
    for src, st, tb, sq in ((b, start_b, table_b, seqs), (a, start, table, later), (b, start_b, table_b, seqs)):
        put(src)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for out in outs:
            check_attention(out[:st[-1]], src, st, tb, sq)


@pytest.mark.gpu
def test_attention_twice_gives_the_same_bits_and_runs_on_side_streams(native_lib):
    from paged_attention import paged_attention

    for seqs in ([(1, 1 + (i * 977) % 3001) for i in range(30)], [(300, 1000), (1, 2000), (90, 90)]):
        a, start, table = build(seqs, seed=6)
        first = paged_attention(**a)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([paged_attention(**a) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(first, o) for group in outs for o in group)


# ------------------------------------------------------------------ append on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,table", [(BF, BF), (BF, F32), (HF, HF), (HF, F32)])
@pytest.mark.parametrize("N,heads,dim,page", [(1, (12, 2), 128, 16), (3, (4, 4), 16, 7), (64, (12, 2), 128, 16), (257, (14, 2), 64, 48), (40, (0, 3), 128, 64)])
def test_append(native_lib, dtype, table, N, heads, dim, page):
    """y = a cos -+ b sin in fp32: half a step of the result, and three fp32 roundings of at most |a cos| + |b sin|."""
    from paged_attention import paged_append

    Hq, Hkv = heads
    wide = gen((N, (Hq + 2 * Hkv) * dim), dtype, 1).cuda()
    q, k, v = (t.unflatten(1, (-1, dim)) if t.shape[1] else None for t in wide.split([Hq * dim, Hkv * dim, Hkv * dim], 1))
    cos, sin = gen((N, dim), table, 2).cuda(), gen((N, dim), table, 3).cuda()
    n_pages = -(-2 * N // page) + 1
    kp, vp = gen((n_pages, Hkv, page, dim), dtype, 4).cuda(), gen((n_pages, page, Hkv, dim), dtype, 5).cuda().transpose(1, 2).contiguous()
    slots = torch.randperm(n_pages * page, generator=torch.Generator().manual_seed(6))[:N].cuda()
    if N > 2:
        slots[1], slots[2] = -1, n_pages * page   # padding
    k0, v0 = kp.clone(), vp.clone()
    got = paged_append(q, k, v, cos, sin, kp, vp, slots)
    c, s = cos.double()[:, None], sin.double()[:, None]

    def turned(x):
        x = x.double()
        return x * c + torch.cat([-x[..., dim // 2:], x[..., :dim // 2]], -1) * s, (x * c).abs() + (torch.cat([x[..., dim // 2:], x[..., :dim // 2]], -1) * s).abs()

    half = torch.finfo(dtype).eps / 2

    def near(x, want, size):
        tol = half * want.abs() * 1.001 + 3 * 2 ** -24 * size + (2 ** -25 if dtype == HF else 0)
        assert ((x.double() - want).abs() <= tol).all()

    if Hq:
        near(got, *turned(q))
    else:
        assert got is None
    ok = (slots >= 0) & (slots < n_pages * page)
    at = slots[ok]
    want, size = turned(k)
    near(kp[at // page, :, at % page], want[ok], size[ok])
    v0[at // page, :, at % page] = v[ok]
    assert torch.equal(vp, v0)
    k0[at // page, :, at % page] = kp[at // page, :, at % page]
    assert torch.equal(kp, k0)   # no other row has changed


@pytest.mark.gpu
def test_append_without_rotation_in_place_and_with_rows_first_pages(native_lib):
    from paged_attention import paged_append

    q, k, v = gen((5, 4, 64), seed=1).cuda(), gen((5, 2, 64), seed=2).cuda(), gen((5, 2, 64), seed=3).cuda()
    kp, vp = (torch.zeros(3, 16, 2, 64, dtype=BF, device="cuda").transpose(1, 2) for _ in range(2))
    slots = torch.tensor([3, 17, 40, 0, 47], device="cuda")
    got = paged_append(q, k, v, None, None, kp, vp, slots)
    assert torch.equal(got, q)
    for x, p in ((k, kp), (v, vp)):
        assert torch.equal(p.transpose(1, 2).reshape(48, 2, 64)[slots], x)
    cos, sin = gen((5, 64), F32, 4).cuda(), gen((5, 64), F32, 5).cuda()
    want = paged_append(q, k, v, cos, sin, kp, vp, slots)
    same = paged_append(q, k, v, cos, sin, kp, vp, slots, q_out=q)
    assert same is q and torch.equal(q, want)


# ------------------------------------------------------------------ the draw on the GPU
def logits_like(rows, cols, dtype, seed, spread=2.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * spread
    x += (torch.rand(rows, cols, generator=g) < 200.0 / cols) * (4 - 3 * torch.rand(rows, cols, generator=g).log())
    return x.to(dtype)


def check_draw(x, u, **settings):
    from sampling import sample_rows

    dev = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else F32).cuda() if v is not None else None for k, v in settings.items()}
    got = sample_rows(x.cuda(), torch.as_tensor(u, dtype=F32).cuda(), **dev).tolist()
    host = {k: None if v is None else dev[k].cpu().numpy().astype(np.float64) for k, v in settings.items()}
    want = ref.draw(x.double().numpy(), np.float32(u).astype(np.float64), **host)
    assert got == want, [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b][:5]


# A token differs from the 64-bit one only where u falls between a boundary and where the weights' errors have moved it.  Tokens with t < 12 (temperature 1) are off
# by 2^-31 of the row's maximum, the others by 2^-22 of themselves, as good as independent: behind the first ones every boundary has moved by some 2^-31 of the sum,
# 151936 of them make 7e-5 of the draws from a row without filters; for n like tokens boundary i moves by sqrt(i) 2^-22 weights, 6e-5 of the draws.  Rows cut to a
# list have a few hundred boundaries, 1e-6.  All rows below together: less than one run in ten; the seeds are fixed.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("cols", [1, 2, 7, 100, 1000, 4097, 33000, 151936])
def test_draw(native_lib, dtype, cols):
    rows = 12
    x = logits_like(rows, cols, dtype, cols)
    r = np.random.default_rng(cols)
    u, T, k, p, m = r.random(rows), r.uniform(0.5, 1.5, rows), r.integers(1, 400, rows), r.uniform(0.3, 1.0, rows), r.uniform(0.001, 0.2, rows)
    check_draw(x, u)
    check_draw(x, u, temperature=T)
    check_draw(x, u, temperature=T, top_k=k)
    check_draw(x, u, temperature=T, top_p=p)
    check_draw(x, u, temperature=T, min_p=m)
    check_draw(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    check_draw(x, u, top_k=np.full(rows, cols // 2 + 1), top_p=p)
    check_draw(x, u, temperature=np.full(rows, 5.0), top_p=np.full(rows, 0.95))   # half of the vocabulary and more
    check_draw(x, u, temperature=np.zeros(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cols", [(BF, 5000), (F32, 5000), (BF, 151936), (F32, 60000)])
def test_draw_with_lists_around_every_size(native_lib, dtype, cols):
    """Lists that fill a warp, a run, a round of the CTA's threads, or a token more: in one CTA per row and in several."""
    k = [1, 2, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049]
    rows = len(k)
    x = logits_like(rows, cols, dtype, 7 + cols)
    u = np.random.default_rng(cols).random(rows)
    check_draw(x, u, top_k=np.array(k))
    check_draw(x, u, top_k=np.array(k), temperature=np.full(rows, 1.7), top_p=np.full(rows, 0.97))
    check_draw(x.repeat(7, 1), np.tile(u, 7), top_k=np.tile(k, 7))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_draw_from_the_longest_row(native_lib, dtype):
    """4194304 - 1 like tokens of weight w and a larger one of weight 1: u times the sum lies (u N w + u - 1) / w tokens behind the larger one, which an error of
    2^-22 in w moves by 1e-7 of a token."""
    x = torch.zeros(2, 1 << 22, dtype=dtype)
    x[:, 1234567] = 10.0
    u, hot = np.array([0.1, 0.77]), np.full(2, 100.0)
    check_draw(x, u, temperature=hot)
    check_draw(x, u, temperature=hot, top_k=np.array([1000000, 3]))
    check_draw(x, u, temperature=hot, min_p=np.array([0.5, 0.95]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_draw_settings_of_each_row(native_lib, dtype):
    rows, cols = 64, 20000
    x = logits_like(rows, cols, dtype, 1)
    r = np.random.default_rng(2)
    u = r.random(rows)
    on = lambda v, off: np.where(r.random(rows) < 0.5, v, off)
    check_draw(x, u, temperature=on(r.uniform(0.5, 1.5, rows), 0.0), top_k=on(r.integers(1, 2000, rows), 0), top_p=on(r.uniform(0.3, 1, rows), 1.0),
               min_p=on(r.uniform(0.001, 0.2, rows), 0.0))
    check_draw(x, u, temperature=np.full(rows, 1e-6), top_k=np.full(rows, 1 << 30), top_p=np.full(rows, 2.0), min_p=np.full(rows, -1.0))
    check_draw(x, u, temperature=np.full(rows, 1e4), top_k=np.full(rows, 700))
    for edge in (0.0, 1.0 - 2.0 ** -24):
        check_draw(x, np.full(rows, edge), top_k=on(r.integers(1, 2000, rows), 0), top_p=on(r.uniform(0.3, 1, rows), 1.0))
    check_draw(x, u, top_p=np.zeros(rows))                      # the first always stays
    check_draw(x, u, top_p=np.full(rows, 1e-30))
    check_draw(x, u, min_p=np.ones(rows))                       # equals of the maximum
    check_draw(x, u, min_p=np.full(rows, 3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [5, 1000, 151936])
def test_draw_of_equal_masked_and_odd_values(native_lib, cols):
    """Ties go to the lowest index, at the border of top-k and of top-p alike; masked, infinite and NaN logits."""
    r = np.random.default_rng(cols)
    rows, inf = 16, float("inf")
    u = np.float32(r.integers(0, 1 << 20, rows)) / (1 << 20)
    k = r.integers(1, cols + 1, rows)
    few = torch.tensor(r.integers(0, 3, (rows, cols)), dtype=F32)          # weights 1, e^-1, e^-2 in thousands
    flat = torch.zeros(rows, cols)
    # (borders that fall on a multiple of a weight: sums of ones and powers of two are exact, here and there)
    check_draw(flat, u, top_k=k)
    check_draw(flat, u, top_p=np.full(rows, 0.5))
    check_draw(flat, u, top_k=k, top_p=np.full(rows, 0.25), min_p=np.ones(rows))
    check_draw(few, u, top_k=k)
    check_draw(few, u, top_k=k, top_p=r.uniform(0.2, 0.9, rows))
    masked = few.clone()
    masked[:, ::2] = -inf
    check_draw(masked, u, top_k=k)
    check_draw(masked, u, top_p=r.uniform(0.2, 0.9, rows))
    odd = few.clone()
    odd[3, 1] = odd[7, cols - 1] = float("nan")     # rows with a NaN have nothing to draw from
    odd[1::3, 2] = inf
    odd[1::3, 4] = inf
    odd[2::3, :] = -inf
    odd[5] = float("nan")
    odd[8, 3] = -0.0
    odd[11] = -0.0
    odd[11, 2] = 0.0
    odd[14] = torch.finfo(F32).min
    for settings in ({}, {"top_k": k}, {"top_p": np.full(rows, 0.7)}, {"temperature": np.zeros(rows)}, {"min_p": np.full(rows, 0.3)}):
        check_draw(odd, u, **settings)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cols,rows", [(BF, 151936, 6), (F32, 151936, 70), (F32, 400001, 5), (HF, 700001, 3), (BF, 30011, 200)])
def test_draw_from_more_than_a_list_holds(native_lib, dtype, cols, rows):
    """Thousands of tokens kept, borders within thousands of equal logits, rows that do not fit into shared memory or start anywhere."""
    x = logits_like(rows, cols, dtype, 3, spread=1.0)
    r = np.random.default_rng(4)
    u = r.random(rows)
    for k in (2047, 2048, 2049, 5000, 20000):
        check_draw(x, u, top_k=np.full(rows, k), temperature=np.full(rows, 2.0))
    check_draw(x, u, temperature=np.full(rows, 3.0), top_p=r.uniform(0.5, 0.999, rows))
    check_draw(x, u, temperature=np.full(rows, 3.0), top_p=r.uniform(0.5, 0.999, rows), top_k=r.integers(1, 30000, rows), min_p=np.full(rows, 1e-4))
    coarse = (x.float() / 4).round().to(dtype)      # a handful of different values
    check_draw(coarse, u, top_k=r.integers(1, cols, rows))
    check_draw(coarse, u, top_k=r.integers(1, cols, rows), temperature=np.full(rows, 2.0), top_p=r.uniform(0.5, 0.999, rows))


@pytest.mark.gpu
def test_draw_strides_captures_and_numbers_out_of_range(native_lib):
    from sampling import sample_rows

    wide = logits_like(6, 3001, BF, 9).cuda()
    x = wide[:, 3:2998]   # rows that start anywhere
    u = torch.rand(6, generator=torch.Generator().manual_seed(1)).cuda()
    p = torch.full((6,), 0.9).cuda()
    want = ref.draw(x.double().cpu().numpy(), u.double().cpu().numpy(), top_p=p.double().cpu().numpy())
    assert sample_rows(x, u, top_p=p).tolist() == want
    static_u, out = u.clone(), torch.zeros(6, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_rows(x, static_u, top_p=p, out=out)
    for seed in (2, 3):
        static_u.copy_(torch.rand(6, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        assert out.tolist() == ref.draw(x.double().cpu().numpy(), static_u.double().cpu().numpy(), top_p=p.double().cpu().numpy())
    low, high = sample_rows(x, torch.full_like(u, -1.0)), sample_rows(x, torch.full_like(u, 2.0))
    nan = sample_rows(x, torch.full_like(u, float("nan")))
    assert (low == 0).all() and (nan == 0).all() and (high == x.shape[1] - 1).all()
    many = logits_like(3000, 50, F32, 4)
    check_draw(many, np.random.default_rng(0).random(3000), top_k=np.full(3000, 9))


@pytest.mark.gpu
def test_serving_steps_of_two_layers(native_lib):
    """Prompts in pieces, then decoding, two sequences that come and one that goes, through two layers of append -> attention, drawn tokens at the end of
    each step: every step's result against the operators' statements on the whole history."""
    from paged_attention import PagedKVCache
    from sampling import Sampler

    Hq, Hkv, D, V = 4, 2, 64, 500
    cache = PagedKVCache(40, 16, 2, Hkv, D)
    table = gen((V, (Hq + 2 * Hkv) * D), seed=1).cuda()      # a token's q, k and v of layer 0
    head = gen((Hq * D, V), seed=2, scale=0.3).cuda()
    mix = gen((Hq * D, (Hq + 2 * Hkv) * D), seed=3, scale=0.06).cuda()
    inv = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    sampler = Sampler(temperature=0.7, top_k=40, top_p=0.9, seed=5)
    seqs = {cache.open(): list(range(37)), cache.open(): [9, 8, 7]}
    done = {s: 0 for s in seqs}
    hist = {}   # (layer, seq) -> rotated keys and values so far
    for turn in range(6):
        if turn == 3:
            first = next(iter(seqs))
            cache.close(first)
            del seqs[first]
            s = cache.open()
            seqs[s], done[s] = list(range(100, 150)), 0
        take = {s: min(20, len(t) - done[s]) for s, t in seqs.items()}
        st = cache.step(list(seqs), list(take.values()))
        ids = torch.tensor([x for s, t in seqs.items() for x in t[done[s]:done[s] + take[s]]], device="cuda")
        angle = (st.positions.double().cpu()[:, None] * inv).repeat(1, 2)
        cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        qkv = table[ids]
        for layer in range(2):
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
            rotated = cache.append(layer, st, q, k, v, cos, sin)
            out = cache.attend(layer, st, rotated)
            # the statement: this step's rows behind those of the steps before
            kk = cache.k[layer].transpose(1, 2).reshape(-1, Hkv, D)[st.slots].cpu()
            half = torch.finfo(BF).eps / 2
            x, c, sn = k.double().cpu(), cos.double().cpu()[:, None], sin.double().cpu()[:, None]
            turned = x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * sn
            size = (x * c).abs() + (torch.cat([x[..., D // 2:], x[..., :D // 2]], -1) * sn).abs()
            assert ((kk.double() - turned).abs() <= half * turned.abs() * 1.001 + 3 * 2 ** -24 * size).all()
            at, pages, vpages, tab = 0, [], [], []
            for s, n in take.items():
                old = hist.get((layer, s), (torch.zeros(0, Hkv, D, dtype=BF),) * 2)
                new = torch.cat([old[0], kk[at:at + n]]), torch.cat([old[1], v[at:at + n].cpu()])
                hist[layer, s] = new
                tab.append([len(pages) + i for i in range(-(-len(new[0]) // 16))])
                for i in range(0, len(new[0]), 16):
                    for store, rows in ((pages, new[0]), (vpages, new[1])):
                        store.append(torch.nn.functional.pad(rows[i:i + 16], (0, 0, 0, 0, 0, 16 - len(rows[i:i + 16]))).transpose(0, 1))
                at += n
            lens = [(take[s], done[s] + take[s]) for s in seqs]
            check_attention(out, {"q": rotated, "k_pages": torch.stack(pages), "v_pages": torch.stack(vpages)}, st.q_start.tolist(), tab, lens)
            qkv = qkv + out.flatten(1) @ mix
        tokens = sampler((out.flatten(1) @ head)[st.last])
        assert tokens.shape == (len(seqs),) and ((tokens >= 0) & (tokens < V)).all()
        for s, tok in zip(seqs, tokens.tolist()):
            done[s] += take[s]
            if done[s] == len(seqs[s]):
                seqs[s].append(tok)
    for s in list(seqs):
        cache.close(s)
    assert cache.free_pages == 40


@pytest.mark.gpu
def test_attention_without_the_tensor_core_kernels(native_lib):
    """B200NN_DISABLE_TC5=1 takes another kernel for every shape; the switch is read once, so in a process of its own."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    tests = Path(__file__).resolve().parent
    code = ("import sys; sys.path[:0] = [r'%s', r'%s']\n"
            "import test_paged_and_sampling as t\n"
            "from paged_attention import paged_attention\n"
            "for name in ('empty_and_short', 'decode_d64', 'decode_window', 'draft_4', 'chunk_window', 'chunk_odd'):\n"
            "    case = t.CASES[name]\n"
            "    a, start, table = t.build(**case)\n"
            "    t.check_attention(paged_attention(**a, window=case.get('window', 0)), a, start, table, case['seqs'], case.get('window', 0))\n"
            "print('done')\n") % (tests, tests.parent / "pytorch-apple_b200")
    res = subprocess.run([sys.executable, "-c", code], env={**os.environ, "B200NN_DISABLE_TC5": "1"}, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "done" in res.stdout, res.stderr[-2000:]
