"""Group-rollout operators on the CPU: what they refuse, and their plain paths
(shared-prefix decode attention, cache-page copies, RMSNorm with an fp8 output)."""

import math

import pytest
import torch

from rl_b200.ops.attention import paged_decode_attention_ref, shared_prefix_decode_attention
from rl_b200.ops.cache_pages import copy_cache_pages
from rl_b200.ops.norm import add_rms_norm_fp8, rms_norm_fp8


def _attn_inputs(B=3, nq=4, nkv=2, hd=8, bs=4, width=3):
    g = torch.Generator().manual_seed(0)
    kc = torch.randn(B * width + 1, bs, nkv, hd, generator=g)
    vc = torch.randn(B * width + 1, bs, nkv, hd, generator=g)
    bt = torch.arange(B * width, dtype=torch.int32).view(B, width) + 1
    return torch.randn(B, nq, hd, generator=g), kc, vc, bt


def test_shared_prefix_attention_is_paged_attention_of_complete_tables():
    q, kc, vc, bt = _attn_inputs()
    lens = torch.tensor([12, 0, 5], dtype=torch.int32)
    starts, prefix = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    out = shared_prefix_decode_attention(q, kc, vc, bt, lens, starts, prefix)
    ref = paged_decode_attention_ref(q[[0, 2]], kc, vc, bt[[0, 2]], lens[[0, 2]])
    assert torch.equal(out[[0, 2]], ref) and not out[1].any()
    # fp8 caches are dequantised with their scales
    k8, v8 = (kc / 0.02).clamp(-448, 448).to(torch.float8_e4m3fn), (vc / 0.02).clamp(-448, 448).to(torch.float8_e4m3fn)
    o8 = shared_prefix_decode_attention(q, k8, v8, bt, lens, starts, prefix, k_scale=0.02, v_scale=0.02)
    r8 = paged_decode_attention_ref(q[:1], k8.float() * 0.02, v8.float() * 0.02, bt[:1], lens[:1], 1 / math.sqrt(8))
    assert torch.equal(o8[:1], r8)


@pytest.mark.parametrize("change", ["starts_len", "starts_dtype", "lens_dim", "tables_rows", "heads", "head_dim",
                                    "v_shape", "q_dim", "lens_count"])
def test_shared_prefix_attention_refuses(change):
    q, kc, vc, bt = _attn_inputs()
    a = dict(q=q, k_cache=kc, v_cache=vc, block_tables=bt, seq_lens=torch.tensor([12, 3, 5], dtype=torch.int32),
             group_starts=torch.tensor([0, 3], dtype=torch.int32), prefix_lens=torch.tensor([3], dtype=torch.int32))
    shared_prefix_decode_attention(**a)
    a.update({"starts_len": {"group_starts": torch.tensor([0, 2, 3], dtype=torch.int32)},
              "starts_dtype": {"group_starts": torch.tensor([0.0, 3.0])},
              "lens_dim": {"seq_lens": torch.tensor([[12, 3, 5]], dtype=torch.int32)},
              "tables_rows": {"block_tables": bt[:2]},
              "heads": {"q": q[:, :3]},
              "head_dim": {"q": q[..., :4]},
              "v_shape": {"v_cache": vc[:4]},
              "q_dim": {"q": q[0]},
              "lens_count": {"seq_lens": torch.tensor([12, 3], dtype=torch.int32)}}[change])
    with pytest.raises(ValueError):
        shared_prefix_decode_attention(**a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
def test_copy_cache_pages(dtype):
    cache = torch.randn(3, 2, 7, 4, 2, 5).to(dtype)
    want = cache.float()
    want[:, :, 5] = want[:, :, 1]
    want[:, :, 6, :2] = want[:, :, 1, :2]
    want[:, :, 0, :1] = want[:, :, 2, :1]
    copy_cache_pages(cache, [1, 1, 2, 3], torch.tensor([5, 6, 0, 4]), [4, 2, 1, 0])
    assert torch.equal(cache.float(), want)
    copy_cache_pages(cache, [], [])
    assert torch.equal(cache.float(), want)
    copy_cache_pages(cache, [6], [0])  # whole pages without token counts
    want[:, :, 0] = want[:, :, 6]
    assert torch.equal(cache.float(), want)


@pytest.mark.parametrize("src,dst,tokens,error", [
    ([1], [7], None, IndexError), ([-1], [2], None, IndexError), ([1], [2], [5], ValueError),
    ([1], [2], [-1], ValueError), ([1, 3], [2, 2], None, ValueError), ([1, 2], [2, 3], None, ValueError),
    ([1], [1], None, ValueError), ([1, 2], [3], None, ValueError), ([1], [3], [1, 1], ValueError),
    (torch.tensor([1.0]), [2], None, ValueError), (torch.tensor([[1]]), [2], None, ValueError)])
def test_copy_cache_pages_refuses(src, dst, tokens, error):
    cache = torch.randn(2, 2, 7, 4, 2, 4)
    before = cache.clone()
    with pytest.raises(error):
        copy_cache_pages(cache, src, dst, tokens)
    assert torch.equal(cache, before)


def test_copy_cache_pages_refuses_strided_caches():
    with pytest.raises(ValueError):
        copy_cache_pages(torch.zeros(2, 2, 7, 4, 2, 8)[..., :4], [1], [2])
    with pytest.raises(ValueError):
        copy_cache_pages(torch.zeros(7, 4, 2), [1], [2])


@pytest.mark.parametrize("mx", [True, False])
def test_norm_fp8_is_norm_then_quantisation(mx):
    from rl_b200.ops.fp8_gemm import fp8_linear, fp8_linear_mx, fp8_linear_quantised, mx_weight_scales
    from rl_b200.ops.norm import add_rms_norm, rms_norm
    from rl_b200.ops.quant import quant_fp8_block

    g = torch.Generator().manual_seed(0)
    x, d = (torch.randn(2, 3, 256, generator=g, dtype=torch.float32).bfloat16() for _ in range(2))
    w = torch.ones(256).bfloat16()
    w_q, w_s = quant_fp8_block(torch.randn(40, 256, generator=g), 128, mx)
    w_s = mx_weight_scales(w_s) if mx else w_s
    linear = fp8_linear_mx if mx else fp8_linear
    q, sc, s = add_rms_norm_fp8(x, d, w, mx=mx)
    h, s_ref = add_rms_norm(x, d, w)
    assert torch.equal(s, s_ref) and q.shape == x.shape and q.dtype == torch.float8_e4m3fn
    assert torch.equal(fp8_linear_quantised(q, sc, w_q, w_s, mx), linear(h, w_q, w_s))
    q, sc = rms_norm_fp8(x, w, mx=mx)
    assert torch.equal(fp8_linear_quantised(q, sc, w_q, w_s, mx), linear(rms_norm(x, w), w_q, w_s))


def test_norm_fp8_refuses():
    x, w = torch.zeros(2, 256), torch.ones(256)
    for args in ((torch.zeros(2, 200), torch.ones(200)), (x, torch.ones(128)), (x, w.double())):
        with pytest.raises(ValueError):
            rms_norm_fp8(*args)
    with pytest.raises(ValueError):
        add_rms_norm_fp8(x, torch.zeros(3, 256), w)
    with pytest.raises(ValueError):
        add_rms_norm_fp8(x, x.bfloat16(), w)
    with pytest.raises(RuntimeError):
        rms_norm_fp8(x.requires_grad_(True), w)
    with torch.no_grad():
        rms_norm_fp8(x, w)


# ------------------------------------------------------------------------ rollout engine
def _worker(mg: dict):
    from rl_b200.models.config import get_model_config
    from rl_b200.models.policy.worker import PolicyWorker
    from rl_b200.parallel.state import single_process_state

    pcfg = {"max_total_sequence_length": 96, "precision": "float32", "train_global_batch_size": 12,
            "generation": {"temperature": 1.0, "max_new_tokens": 12,
                           "mcore_generation_config": {"block_size_tokens": 16, **mg}}}
    return PolicyWorker(pcfg, model_cfg=get_model_config("tiny-llama"),
                        pstate=single_process_state(torch.device("cpu")), seed=3)


def _batch(order=None):
    from rl_b200.distributed.batched_data_dict import BatchedDataDict

    g = torch.Generator().manual_seed(0)
    lens = torch.tensor([5, 32, 40, 17]).repeat_interleave(3)
    ids = torch.randint(0, 512, (4, 40), generator=g).repeat_interleave(3, 0)
    order = torch.arange(12) if order is None else order
    return BatchedDataDict({"input_ids": ids[order], "input_lengths": lens[order]})


@pytest.mark.parametrize("order", [None, [0, 3, 1, 6, 7, 4, 5, 8, 9, 2, 11, 10]])
def test_shared_prompt_rollout_equals_copied_prompts(order):
    data = _batch(None if order is None else torch.tensor(order))
    ref = _worker({}).generate(data, greedy=True)
    w = _worker({"enable_shared_prefix_attention": True})
    out = w.generate(data, greedy=True)
    assert torch.equal(out["output_ids"], ref["output_ids"])
    torch.testing.assert_close(out["logprobs"], ref["logprobs"], atol=1e-5, rtol=0)
    assert w.engine._prompts is not None
    starts, lens = w.engine._prefix_groups()
    if order is None:
        assert starts.tolist() == [0, 3, 6, 9, 12] and lens.tolist() == [5, 32, 40, 17]
    assert w.engine._prefix_groups(width=3)[0].tolist() == [3 * s for s in starts.tolist()]
    out_starts, out_lens = torch.full((14,), 77, dtype=torch.int32), torch.full((13,), 77, dtype=torch.int32)
    w.engine._prefix_groups(torch.tensor([0, 1, 5, 11]), out=(out_starts, out_lens))
    assert out_starts[-1] == 4 and out_lens[-1] == 0 and (out_starts.diff() >= 0).all()


def test_rollout_without_duplicates_does_not_share():
    w = _worker({"enable_shared_prefix_attention": True})
    data = _batch(torch.tensor([0, 3, 6, 9]))
    ref = _worker({}).generate(data, greedy=True)
    assert torch.equal(w.generate(data, greedy=True)["output_ids"], ref["output_ids"])
    assert w.engine._prompts is None


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_shared_prompt_speculative_rollout(kv):
    """Speculative decoding over forked prompts (a small LM drafts; target and draft share pages), and an
    fp8 cache: greedy rollouts are those of copied prompts."""
    import dataclasses

    from rl_b200.models.config import get_model_config
    from rl_b200.models.transformer import TransformerLM

    outs = []
    for mg in ({}, {"enable_shared_prefix_attention": True}):
        w = _worker(mg)
        w.engine.kv_dtype = torch.float8_e4m3fn if kv == "fp8" else w.engine.kv_dtype
        draft = TransformerLM(dataclasses.replace(get_model_config("tiny-llama"), num_layers=1),
                              device=torch.device("cpu"), dtype=torch.float32, seed=9)
        w.engine.set_draft(draft, 3)
        outs.append(w.generate(_batch(), greedy=True)["output_ids"])
        assert w.engine.spec_stats["rounds"] > 0
    assert torch.equal(outs[0], outs[1])


def test_shared_prompt_rollout_rules():
    """Which models may attend to shared prompts, and when it pays (the rules of the GPU path)."""
    from types import SimpleNamespace as Heads

    eng = _worker({"enable_shared_prefix_attention": True}).engine
    eng.model, eng.draft, eng.draft_kind = Heads(hd=128, nq=32, nkv=8), Heads(hd=64, nq=8, nkv=2), "lm"
    eng._check_shared_heads(True)
    for bad in (Heads(hd=96, nq=8, nkv=8), Heads(hd=64, nq=130, nkv=2)):
        eng.draft = bad
        eng._check_shared_heads(False)  # the draft is not called
        with pytest.raises(ValueError, match="draft"):
            eng._check_shared_heads(True)
        eng.draft_kind = "eagle3"  # attends on its own
        eng._check_shared_heads(True)
        eng.draft_kind, eng.model, model = "lm", bad, eng.model
        with pytest.raises(ValueError, match="model"):
            eng._check_shared_heads(False)
        eng.model = model
    # 2 x 8 x 128 values of 2 bytes a key: 10 keys saved of a prompt of 10 tokens for two rows
    eng.kv_dtype, eng.num_spec = torch.bfloat16, 3
    eng.shared_prefix_min_bytes = 10 * 2 * 8 * 128 * 2
    assert eng._shared_prefix_pays([0], [10, 10], False)
    assert not eng._shared_prefix_pays([0], [9, 9], False)
    assert eng._shared_prefix_pays([0], [10] * 4096, False) and not eng._shared_prefix_pays([0], [10] * 4097, False)
    assert eng._shared_prefix_pays([0], [10] * 1024, True) and not eng._shared_prefix_pays([0], [10] * 1025, True)


def test_shared_prompt_runs():
    """What decode saves is counted by runs: rows of one prompt that lie apart share nothing."""
    eng = _worker({"enable_shared_prefix_attention": True}).engine
    assert eng._run_starts([0, 0, 1, 1, 0]) == [0, 2, 4] and eng._run_starts([0, 1, 0, 1]) == [0, 1, 2, 3]
    eng.shared_prefix_min_bytes = 1
    assert eng._shared_prefix_pays(eng._run_starts([0, 0, 1, 1]), [9] * 4, False)
    assert not eng._shared_prefix_pays(eng._run_starts([0, 1, 0, 1]), [9] * 4, False)


def test_heads_that_row_by_row_attention_lacks():
    """Query heads per KV head decide whether attention by prompts is a choice (the rule of the GPU path)."""
    from types import SimpleNamespace as Heads

    eng = _worker({"enable_shared_prefix_attention": True}).engine
    eng.draft, eng.draft_kind, eng.num_spec = Heads(hd=128, nq=8, nkv=1), "lm", 3
    for nq, nkv, row_by_row in ((32, 8, True), (8, 8, True), (64, 8, True), (28, 4, False), (12, 2, False), (5, 1, False)):
        eng.model = Heads(hd=128, nq=nq, nkv=nkv)
        assert eng._row_by_row_heads(False) == eng._row_by_row_heads(True) == row_by_row
    eng.model, eng.draft = Heads(hd=128, nq=8, nkv=1), Heads(hd=128, nq=28, nkv=4)
    assert eng._row_by_row_heads(False) and not eng._row_by_row_heads(True)
    eng.draft_kind = "eagle3"  # attends on its own
    assert eng._row_by_row_heads(True)
    assert eng._fits_plan(4096, False) and not eng._fits_plan(4097, False)
    assert eng._fits_plan(1024, True) and not eng._fits_plan(1025, True)


def test_rows_that_are_left_share_where_it_pays_for_them():
    eng = _worker({"enable_shared_prefix_attention": True}).engine
    assert not eng._shares_prompts(torch.arange(4))  # no shared prompts
    eng._prompts = (torch.tensor([0, 0, 0, 1, 1, 2, 0]), torch.tensor([10, 20, 30]))
    token = 2 * eng.model.nkv * eng.model.hd * torch.empty((), dtype=eng.kv_dtype).element_size()
    for limit, rows, shares in ((40, range(7), True), (41, range(7), False), (20, [0, 1, 2], True), (21, [0, 1, 2], False),
                                (20, [2, 3, 4], True), (1, [0, 3, 5, 6], False), (10, [0, 1, 5], True), (1, [2], False)):
        eng.shared_prefix_min_bytes = limit * token
        assert eng._shares_prompts(torch.tensor(list(rows))) == shares
    eng._only_by_prompts = True
    assert eng._shares_prompts(torch.tensor([2]))


@pytest.mark.parametrize("dtype,hd,nkv,rows,limit", [
    (torch.bfloat16, 128, 8, 16, 100 << 20), (torch.bfloat16, 64, 8, 256, 272 << 20), (torch.bfloat16, 64, 2, 16, 83 << 20),
    (torch.float8_e4m3fn, 128, 8, 16, 40 << 20), (torch.float8_e4m3fn, 64, 8, 256, 40 << 20),
    (torch.bfloat16, 32, 8, 64, 40 << 20)])
def test_shared_prompts_pay_by_type_heads_and_rows(dtype, hd, nkv, rows, limit):
    from types import SimpleNamespace as Heads

    eng = _worker({"enable_shared_prefix_attention": True}).engine
    eng.model, eng.kv_dtype = Heads(hd=hd, nq=4 * nkv, nkv=nkv), dtype
    token = 2 * nkv * hd * dtype.itemsize
    tokens = -(-limit // (token * (rows - 1)))  # of one prompt for all the rows
    assert eng._shared_prefix_pays([0], [tokens] * rows, False)
    assert not eng._shared_prefix_pays([0], [tokens - 1] * rows, False)


@pytest.mark.parametrize("words,has,lacks", [
    ({"shared_prefix_error_flag": 1}, ["group starts"], ["wait expired"]),
    ({"shared_prefix_error_flag": 2}, ["block-table entry"], ["wait expired"]),
    ({"shared_prefix_error_flag": 3}, ["wait expired", "shared_prefix_error_flag"], ["block-table"]),
    ({"shared_prefix_error_flag": 2, "gemm_error_flag": 1}, ["wait expired", "gemm_error_flag", "block-table entry"], [])])
def test_error_words_of_device_data_are_not_called_waits(monkeypatch, words, has, lacks):
    from types import SimpleNamespace

    from rl_b200.ops import _ext

    flags = {name: (lambda reset, v=words.get(name, 0): v) for name in _ext.ERROR_FLAGS}
    monkeypatch.setattr(_ext, "has_ext", lambda: True)
    monkeypatch.setattr(_ext, "ext", lambda: SimpleNamespace(**flags))
    with pytest.raises(_ext.DeviceWaitError) as e:
        _ext.check_device_errors()
    assert all(h in str(e.value) for h in has) and not any(x in str(e.value) for x in lacks)
