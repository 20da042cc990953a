"""Cases of the group-rollout operators: decode attention over a shared prompt, cache-page
copies and the RMSNorm that hands its output to an fp8 projection.

A GRPO step draws many completions of each prompt.  Three operators carry such a group
through a decode step: the pages of its prompt are copied or forked to its rows, every row's
new token attends to the group's prompt (read once for all of them) and to its own tokens, and
the residual stream is added, normalised and quantised for the fp8 projections.

``own`` selects the framework's calls; otherwise ``run`` computes the same outputs with
elementary torch operations in 32 bits.
"""

import random

import torch

own = False

FP8_MAX = 448.0


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the last live group of a batch: 8 completions of one short prompt, just begun (latency)
        _attention("attn_one_group", 1, 8, 128, 16),
        # a GRPO batch of 4 prompts x 16 completions, every completion 1 to 1024 tokens long
        _attention("attn_grpo", 4, 16, 1024, 1024, ragged=True),
        # one long-context prompt and 32 completions of it
        _attention("attn_long_prompt", 1, 32, 32768, 512, ragged=True),
        # the fp8 cache, 8 prompts x 16 completions
        _attention("attn_fp8_cache", 8, 16, 2048, 1024, cache="fp8", ragged=True),
        # 7 query heads per KV head of 64 dims, small pages, groups of uneven size, odd lengths
        _attention("attn_odd", 5, 7, 777, 333, heads=14, kv_heads=2, head_dim=64, block=16, ragged=True),
        # a large rollout batch: 16 prompts x 16 completions
        _attention("attn_large", 16, 16, 2048, 2048, ragged=True),
        # fork: 7 more rows for one prompt whose last page holds 37 tokens
        _copy("fork_tail", 1, 7, 1, 37, layers=16, block=256),
        # every row of a group gets its own copy of the whole prompt (4 prompts x 16 rows)
        _copy("copy_prompts", 4, 15, 4, 200, layers=8, block=256),
        # one sequence decodes: the smallest call
        _norm("norm_one_row", 1, 4096, "row"),
        # a decode step of 64 sequences
        _norm("norm_decode", 64, 4096, "mx"),
        # a batch that fits no tile, narrow rows
        _norm("norm_odd", 333, 1536, "row"),
        # a prefill pass
        _norm("norm_prefill", 16384, 4096, "row"),
    ]


def _attention(name, groups, rows, prefix, suffix, heads=32, kv_heads=8, head_dim=128, block=256, cache="bf16",
               ragged=False):
    return {"name": name, "op": "attention", "groups": groups, "rows": rows, "prefix": prefix, "suffix": suffix,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "cache": cache,
            "ragged": ragged}


def _copy(name, sources, forks, pages, tail, layers, block, kv_heads=8, head_dim=128):
    return {"name": name, "op": "copy", "sources": sources, "forks": forks, "pages": pages, "tail": tail,
            "layers": layers, "block": block, "kv_heads": kv_heads, "head_dim": head_dim}


def _norm(name, rows, hidden, layout):
    return {"name": name, "op": "norm", "rows": rows, "hidden": hidden, "layout": layout}


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "copy", "norm"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        case = _attention("", _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 32), _log_uniform(rng, 1, 16384),
                          _log_uniform(rng, 1, 2048), heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8]),
                          kv_heads=kv_heads, head_dim=rng.choice([64, 128]), block=rng.choice([16, 64, 256]),
                          cache=rng.choice(["bf16", "fp8"]), ragged=rng.random() < 0.75)
        # at most the tokens of the largest listed case
        while case["groups"] * (case["prefix"] + case["rows"] * case["suffix"]) > 400_000:
            case["groups"] = max(1, case["groups"] // 2)
            case["suffix"] = max(1, case["suffix"] // 2)
    elif op == "copy":
        block = rng.choice([16, 64, 256])
        case = _copy("", rng.randint(1, 6), _log_uniform(rng, 1, 15), _log_uniform(rng, 1, 4), rng.randint(1, block),
                     layers=rng.randint(1, 8), block=block, kv_heads=rng.choice([1, 2, 8]),
                     head_dim=rng.choice([64, 128]))
    else:
        case = _norm("", _log_uniform(rng, 1, 16384), 128 * rng.choice([1, 5, 8, 16, 28, 32, 40, 64]),
                     rng.choice(["row", "mx"]))
        while case["rows"] * case["hidden"] > 16384 * 4096 or case["layout"] == "mx" and case["rows"] > 256:
            case["rows"] //= 2
    del case["name"]
    return case


# ----------------------------------------------------------------------------- the lengths
def _lengths(case):
    """(rows per group, prompt tokens per group, completion tokens per row): of the case alone."""
    g, n, p, s = case["groups"], case["rows"], case["prefix"], case["suffix"]
    if not case["ragged"]:
        return [n] * g, [p] * g, [s] * (g * n)
    rng = random.Random(1_000_003 * g + 10_007 * n + 101 * p + s)
    rows = [n] + [rng.randint((n + 1) // 2, n) for _ in range(g - 1)]
    prompts = [p] + [rng.randint((p + 1) // 2, p) for _ in range(g - 1)]
    return rows, prompts, [rng.randint(1, s) for _ in range(sum(rows))]


def _tables(case):
    """Block tables as the engine makes them for a forked group: the full pages of the prompt are shared,
    its last, partly filled page and what follows are the row's own.  (tables, sequence lengths, pages,
    pairs of pages that hold the same prompt tokens)"""
    rows, prompts, suffixes = _lengths(case)
    bs = case["block"]
    tables, lens, twins, page, row = [], [], [], 1, 0  # page 0 is never read
    for n, p in zip(rows, prompts):
        full = p // bs
        shared = list(range(page, page + full))
        page += full
        tail = None
        for _ in range(n):
            total = p + suffixes[row]
            mine = list(range(page, page + -(-total // bs) - full))
            page += len(mine)
            if p % bs:
                tail = mine[0] if tail is None else tail
                if mine[0] != tail:
                    twins.append((tail, mine[0]))
            tables.append(shared + mine)
            lens.append(total)
            row += 1
    width = max(len(t) for t in tables)
    return [t + [0] * (width - len(t)) for t in tables], lens, page, twins


def _pairs(case):
    """(source pages, destination pages, tokens of each): every source's pages to each of its forks."""
    src, dst, tokens, page = [], [], [], 1
    for _ in range(case["sources"]):
        mine = list(range(page, page + case["pages"]))
        page += case["pages"]
        for _ in range(case["forks"]):
            src += mine
            dst += range(page, page + case["pages"])
            tokens += [case["block"]] * (case["pages"] - 1) + [case["tail"]]
            page += case["pages"]
    return src, dst, tokens, page


# ------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    if case["op"] == "attention":
        tables, lens, pages, twins = _tables(case)
        shape = (pages, case["block"], case["kv_heads"], case["head_dim"])
        k, v = normal(*shape), normal(*shape)
        k_scale = v_scale = 1.0
        if case["cache"] == "fp8":
            k_scale, v_scale = 0.0125, 0.01  # calibrated: largest value / 448
            k = (k.float() / k_scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
            v = (v.float() / v_scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
        order = torch.randperm(pages - 1, device="cuda", generator=gen) + 1  # pages lie anywhere in the cache
        place = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), order])
        if twins:
            a, b = (place[torch.tensor(x, device="cuda")] for x in zip(*twins))
            for t in (k.view(torch.uint8), v.view(torch.uint8)):
                t[b] = t[a]  # the forked copy of the prompt's last page
        rows, prompts, _ = _lengths(case)
        starts = torch.tensor([0] + rows).cumsum(0).to("cuda", torch.int32)
        return {"op": "attention", "q": normal(len(lens), case["heads"], case["head_dim"]), "k": k, "v": v,
                "tables": place[torch.tensor(tables, device="cuda")].to(torch.int32),
                "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "starts": starts,
                "prompts": torch.tensor(prompts, dtype=torch.int32, device="cuda"), "k_scale": k_scale,
                "v_scale": v_scale}
    if case["op"] == "copy":
        src, dst, tokens, pages = _pairs(case)
        order = [0] + random.Random(seed).sample(range(1, pages), pages - 1)
        cache = normal(case["layers"] * 2, pages, case["block"], case["kv_heads"], case["head_dim"])
        return {"op": "copy", "cache": cache.view(case["layers"], 2, *cache.shape[1:]),
                "src": [order[i] for i in src], "dst": [order[i] for i in dst], "tokens": tokens}
    h = case["hidden"]
    return {"op": "norm", "x": normal(case["rows"], h), "delta": normal(case["rows"], h, scale=0.5),
            "w": 1 + normal(h, scale=0.1), "eps": 1e-5, "mx": case["layout"] == "mx"}


# -------------------------------------------------------------------------------- the runs
def run(state):
    return {"attention": _run_attention, "copy": _run_copy, "norm": _run_norm}[state["op"]](state)


def _run_attention(s):
    if own:
        from rl_b200.ops.attention import shared_prefix_decode_attention

        return shared_prefix_decode_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["starts"],
                                              s["prompts"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    q, tables, lens = s["q"].float(), s["tables"].long(), s["lens"]
    b, nq, hd = q.shape
    nkv = s["k"].shape[2]
    k = s["k"][tables].flatten(1, 2).float().transpose(1, 2) * s["k_scale"]  # [B, nkv, T, hd]
    v = s["v"][tables].flatten(1, 2).float().transpose(1, 2) * s["v_scale"]
    scores = torch.matmul(q.view(b, nkv, nq // nkv, hd), k.transpose(2, 3)) / hd ** 0.5
    live = torch.arange(k.shape[2], device=q.device) < lens[:, None]
    scores = scores.masked_fill(~live[:, None, None, :], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, v.masked_fill(~live[:, None, :, None], 0.0)) / p.sum(-1, keepdim=True)
    return out.view(b, nq, hd).to(s["q"].dtype)


def _run_copy(s):
    cache = s["cache"]
    if own:
        from rl_b200.ops.cache_pages import copy_cache_pages

        copy_cache_pages(cache, s["src"], s["dst"], s["tokens"])
    else:
        src, dst, tokens = (torch.tensor(s[n], device=cache.device) for n in ("src", "dst", "tokens"))
        live = torch.arange(cache.shape[3], device=cache.device) < tokens[:, None]
        cache[:, :, dst] = torch.where(live[:, :, None, None], cache[:, :, src], cache[:, :, dst])
    return cache.view(torch.int16)  # copies are equal in every bit


def _run_norm(s):
    if own:
        from rl_b200.ops.norm import add_rms_norm_fp8

        q, scales, total = add_rms_norm_fp8(s["x"], s["delta"], s["w"], s["eps"], mx=s["mx"])
        return _norm_outputs(total, q, scales[:, :q.shape[0]].t() if s["mx"] else scales)
    # the sum is rounded where it is stored, and that is what is normalised; the norm is rounded
    # to the type that an unquantised projection would read
    total = (s["x"].float() + s["delta"].float()).to(s["x"].dtype)
    f = total.float()
    y = (f / torch.sqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * s["w"].float()).to(s["x"].dtype).float()
    groups = y.view(y.shape[0], -1, 128)
    scales = groups.abs().amax(-1).clamp_min(1e-12) / FP8_MAX
    if s["mx"]:
        scales = torch.exp2(torch.ceil(torch.log2(scales)))
    q = (groups / scales[..., None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return _norm_outputs(total, q.view_as(y), scales)


def _norm_outputs(total, q, scales):
    # a scale follows the largest norm of its 128 values, which is a bf16 number: it is given as one
    return {"sum": total, "q": q, "scales": scales.to(torch.bfloat16)}


# -------------------------------------------------------------------------- the definition
def exact(case, seed):
    if case["op"] == "copy":
        return None  # nothing is computed
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    x = s["x"].double() + s["delta"].double()
    total = x.to(torch.bfloat16).double()
    rms = (total.square().sum(-1, keepdim=True) / total.shape[1] + s["eps"]).sqrt()
    y = (total / rms * s["w"].double()).to(torch.bfloat16).double()
    q, scales = torch.empty_like(y), []
    for j in range(0, y.shape[1], 128):
        part = y[:, j:j + 128]
        step = part.abs().amax(1, keepdim=True).clamp(min=1e-12) / FP8_MAX
        if s["mx"]:
            mantissa, exponent = torch.frexp(step)
            step = torch.ldexp(torch.ones_like(step), exponent - (mantissa == 0.5).to(exponent.dtype))
        # an e4m3 value has 4 significant bits above 2^-6 and steps of 2^-9 below
        r = part / step
        e = torch.frexp(r)[1].clamp(min=-5)
        unit = torch.ldexp(torch.ones_like(r), e - 4)
        q[:, j:j + 128] = (torch.round(r / unit) * unit).clamp(-FP8_MAX, FP8_MAX)
        scales.append(step)
    return {"sum": x, "q": q, "scales": torch.cat(scales, 1)}


def _exact_attention(case, s):
    """Row by row, token by token of its page list, in 64 bits."""
    b, nq, hd = s["q"].shape
    nkv, bs = case["kv_heads"], case["block"]
    kc, vc = s["k"].reshape(-1, nkv, hd), s["v"].reshape(-1, nkv, hd)
    out = torch.zeros(b, nq, hd, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(s["lens"].tolist()):
        t = torch.arange(n, device=kc.device)
        slots = s["tables"][i].long()[t // bs] * bs + t % bs
        k = kc[slots].double() * s["k_scale"]
        v = vc[slots].double() * s["v_scale"]
        for j in range(nkv):
            heads = slice(j * (nq // nkv), (j + 1) * (nq // nkv))
            weights = torch.softmax(s["q"][i, heads].double() @ k[:, j].T * hd ** -0.5, 1)
            out[i, heads] = weights @ v[:, j]
    return out


# --------------------------------------------------------------------------------- the work
def work(case):
    if case["op"] == "attention":
        rows, prompts, suffixes = _lengths(case)
        tables, lens, _, _ = _tables(case)
        size = 1 if case["cache"] == "fp8" else 2
        keys = sum(prompts) + sum(suffixes)  # each prompt's keys are read once for its group
        qo = 2 * len(lens) * case["heads"] * case["head_dim"] * 2
        return {"bytes": keys * 2 * case["kv_heads"] * case["head_dim"] * size + qo + 4 * len(tables) * len(tables[0]),
                "flops": 4 * sum(lens) * case["heads"] * case["head_dim"]}
    if case["op"] == "copy":
        src, dst, tokens, _ = _pairs(case)
        row = 2 * case["layers"] * 2 * case["kv_heads"] * case["head_dim"]
        reads = sum(dict(zip(src, tokens)).values())
        return {"bytes": row * (reads + sum(tokens)), "flops": 0}
    n, h = case["rows"], case["hidden"]
    return {"bytes": n * h * (2 + 2 + 2 + 1) + 4 * n * (h // 128) + 2 * h, "flops": 8 * n * h}
