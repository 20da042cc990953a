"""Group-rollout kernels against plain 64-bit implementations: shared-prefix decode
attention, cache-page copies, RMSNorm with an fp8 output, and a decode step of them."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from rl_b200.ops import _ext  # noqa: E402
from rl_b200.ops.attention import shared_prefix_decode_attention, shared_prefix_plan  # noqa: E402
from rl_b200.ops.cache_pages import copy_cache_pages  # noqa: E402
from rl_b200.ops.norm import add_rms_norm_fp8, rms_norm_fp8  # noqa: E402

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}


@pytest.fixture(scope="module", autouse=True)
def _need_ext(cuda_device):
    assert _ext.has_ext(), "native extension must be built and loadable on a GPU box"
    yield


# ------------------------------------------------------------- shared-prefix attention
class Batch:
    """Rows of groups in a paged cache whose unused slots hold NaN."""

    def __init__(self, dev, groups, prefix, lens, nq, nkv, hd, bs, fp8=False, share=True, seed=0, alone=(0, 0),
                 pages=None, q_scale=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.nq, self.nkv, self.hd, self.bs, self.fp8 = nq, nkv, hd, bs, fp8
        B = alone[0] + sum(groups) + alone[1]
        assert len(lens) == B
        width = max(1, -(-max(lens) // bs)) + 1
        need = B * width + 1
        pages = max(need, pages or 0)
        kc = torch.full((pages, bs, nkv, hd), float("nan"), dtype=torch.bfloat16, device=dev)
        vc = kc.clone()
        ids = (pages - 1 - torch.randperm(need - 1, generator=torch.Generator().manual_seed(seed))).view(B, width)
        row = alone[0]
        source = list(range(B))  # the row whose prefix this row repeats
        first = {}
        for n, p in zip(groups, prefix):
            for r in range(row, row + n):
                first[r] = p
                source[r] = row if r > row else r
            row += n
        self.k_scale, self.v_scale = (0.0131, 0.0097) if fp8 else (1.0, 1.0)
        rows_k, rows_v = [], []
        for b, n in enumerate(lens):
            k = torch.randn(n, nkv, hd, device=dev, generator=g).bfloat16()
            v = torch.randn(n, nkv, hd, device=dev, generator=g).bfloat16()
            if source[b] != b:
                p = min(first[b], n, lens[source[b]])
                k[:p], v[:p] = rows_k[source[b]][:p], rows_v[source[b]][:p]
                if share:  # whole pages of the prefix are the leader's
                    ids[b, :p // bs] = ids[source[b], :p // bs]
            rows_k.append(k)
            rows_v.append(v)
            for i in range(0, n, bs):
                m = min(bs, n - i)
                kc[ids[b, i // bs], :m], vc[ids[b, i // bs], :m] = k[i:i + m], v[i:i + m]
        if fp8:
            kc = (kc.float() / self.k_scale).clamp(-448, 448).to(torch.float8_e4m3fn)
            vc = (vc.float() / self.v_scale).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.kc, self.vc = kc, vc
        self.tables = ids.to(torch.int32).to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        starts = [alone[0]]
        for n in groups:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=dev)
        self.prefix = torch.tensor(prefix, dtype=torch.int32, device=dev)
        self.q = (torch.randn(B, nq, hd, device=dev, generator=g) * q_scale).bfloat16()

    def run(self, **kw):
        return shared_prefix_decode_attention(self.q, self.kc, self.vc, self.tables, self.lens, self.starts,
                                              self.prefix, k_scale=self.k_scale, v_scale=self.v_scale, **kw)

    def exact(self, scale=None):
        """(result, bound of the error) in 64 bits, row by row.

        Rounding P to the product's type moves the sum of w|v| by half a step of it at most, the output by
        half a bf16 step.  fp32 scores are off by hd * 2^-24 of the sum of |q k|, which moves every weight
        by as much (twice: numerator and sum); sums and rescalings over n keys add n * 2^-23."""
        scale = scale if scale is not None else 1 / math.sqrt(self.hd)
        B = self.q.shape[0]
        out = torch.zeros(B, self.nq, self.hd, dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(out)
        G = self.nq // self.nkv
        for b, n in enumerate(self.lens.tolist()):
            if n == 0:
                continue
            t = torch.arange(n, device=self.q.device)
            slot = self.tables[b].long()[t // self.bs] * self.bs + t % self.bs
            k = self.kc.view(-1, self.nkv, self.hd)[slot].double() * self.k_scale
            v = self.vc.view(-1, self.nkv, self.hd)[slot].double() * self.v_scale
            for j in range(self.nkv):
                h = slice(j * G, (j + 1) * G)
                q = self.q[b, h].double()
                w = torch.softmax(q @ k[:, j].T * scale, -1)
                out[b, h] = w @ v[:, j]
                size = w @ v[:, j].abs()
                dots = (q.abs() @ k[:, j].abs().T * abs(scale)).amax(-1, keepdim=True)
                half_p = 2.0 ** -11 if self.fp8 else 2.0 ** -8
                fp = 2 * (self.hd * 2.0 ** -24 * dots + n * 2.0 ** -23)
                tol[b, h] = size * (half_p + fp) + 2.0 ** -8 * out[b, h].abs() + 1e-30
        return out, tol

    def check(self, got, **kw):
        ref, tol = self.exact(**kw)
        off = (got.double() - ref).abs()
        assert torch.isfinite(got).all()
        worst = (off / tol.clamp_min(1e-300)).max().item()
        assert (off <= tol).all(), f"error is {worst:.2f} times its bound"
        assert _ext.ext().shared_prefix_error_flag(False) == 0


CASES = [  # groups, prefix, lens, nq, nkv, hd, bs
    ([2], [64], [65, 70], 4, 1, 128, 16),
    ([1], [100], [130], 4, 1, 128, 16),                              # one row shares nothing
    ([3], [63], [64, 65, 100], 8, 2, 128, 64),                       # less than a tile
    ([4, 3], [200, 128], [201, 250, 333, 256, 128, 129, 300], 8, 2, 64, 16),
    ([17], [500], list(range(500, 517)), 4, 1, 128, 256),            # two chunks of query rows
    ([5, 0, 2], [130, 7, 1000], [131, 500, 0, 140, 700, 1500, 999], 14, 2, 64, 32),  # a row without keys, no rows
    ([33], [320], [320 + 7 * i for i in range(33)], 12, 4, 32, 8),
    ([9], [256], [300] * 9, 16, 1, 128, 48),                         # pages that end inside a tile
    ([4], [128], [128, 128, 129, 191], 33, 1, 64, 16),               # 33 query heads a KV head, empty suffixes
    ([6], [150], [151, 170, 160, 333, 150, 200], 5, 5, 128, 5),      # no box of keys fits a page of 5
    ([3], [90], [100, 91, 92], 6, 3, 32, 1),
    ([2], [4000], [4100, 4001], 64, 1, 128, 256),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_shared_prefix_attention(cuda_device, case, fp8):
    groups, prefix, lens, nq, nkv, hd, bs = CASES[case]
    b = Batch(cuda_device, groups, prefix, lens, nq, nkv, hd, bs, fp8=fp8, seed=case)
    b.check(b.run())


def test_shared_prefix_attention_rows_outside_groups_and_copied_prefixes(cuda_device):
    b = Batch(cuda_device, [3, 2], [128, 64], [70, 0, 200, 130, 128, 64, 65, 1, 300], 8, 2, 128, 16, share=False,
              alone=(2, 2))
    out = b.run()
    b.check(out)
    assert not out[1].any()


def test_shared_prefix_attention_lengths_of_one_and_no_groups(cuda_device):
    b = Batch(cuda_device, [], [], [1, 1, 2, 0], 4, 4, 128, 16, alone=(4, 0))
    b.check(b.run())
    b = Batch(cuda_device, [2], [0], [0, 0], 4, 4, 128, 16)
    assert not b.run().any()
    assert b.run()[:0].shape == (0, 4, 128)
    z = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    out = shared_prefix_decode_attention(b.q[:0], b.kc, b.vc, b.tables[:0], z, torch.zeros_like(b.starts), b.prefix)
    assert out.shape == (0, 4, 128)


def test_shared_prefix_attention_prefix_longer_than_a_row(cuda_device):
    # the group's prefix is longer than one of its rows: shared up to that row's length
    b = Batch(cuda_device, [4], [1000], [1000, 200, 1100, 129], 8, 2, 128, 16)
    b.check(b.run())


@pytest.mark.parametrize("fp8", [False, True])
def test_shared_prefix_attention_scale_and_large_scores(cuda_device, fp8):
    # peaked softmax (scores of hundreds), and a negative scale
    b = Batch(cuda_device, [5], [192], [193, 220, 250, 300, 192], 8, 2, 64, 16, fp8=fp8, q_scale=40.0)
    b.check(b.run())
    b.check(b.run(scale=-0.05), scale=-0.05)


def test_shared_prefix_attention_tiny_and_huge_queries_on_fp8(cuda_device):
    # rows of q are brought to a common size by powers of two: their own size does not matter
    for q_scale in (2.0 ** -100, 2.0 ** 60):
        b = Batch(cuda_device, [3], [128], [140, 150, 200], 4, 1, 64, 16, fp8=True, q_scale=q_scale)
        s = 0.125 / q_scale
        b.check(b.run(scale=s), scale=s)


def test_shared_prefix_attention_nan_stays_in_its_row(cuda_device):
    b = Batch(cuda_device, [4], [128], [140, 200, 150, 131], 8, 2, 128, 16)
    clean = b.run()
    b.q[2, 3] = float("nan")
    out = b.run()
    assert out[2, 3].isnan().all()
    keep = torch.ones(4, 8, dtype=torch.bool)
    keep[2, 3] = False
    assert torch.equal(out[keep], clean[keep])
    # a key that is infinite in the shared prefix reaches every row of its head
    b.q[2, 3] = 1.0
    b.kc[b.tables[0, 2], 5, 1, 7] = float("inf")
    out = b.run()
    assert out[:, 4:].isnan().any(-1).any() and torch.equal(out[0, :4], clean[0, :4])


def test_shared_prefix_attention_strided_queries_and_int64_indices(cuda_device):
    b = Batch(cuda_device, [3], [64], [65, 100, 99], 8, 2, 128, 16)
    ref = b.run()
    qkv = torch.zeros(3, 12, 128, dtype=torch.bfloat16, device=cuda_device)
    qkv[:, :8] = b.q
    q0 = b.q
    b.q = qkv[:, :8]  # rows of a QKV projection
    assert torch.equal(b.run(), ref)
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(3, 8, 128)
    odd.copy_(q0)
    b.q = odd
    assert torch.equal(b.run(), ref)
    b.q = q0.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(b.run(), ref)
    b.q, b.tables, b.lens, b.starts = q0, b.tables.long(), b.lens.long(), b.starts.long()
    assert torch.equal(b.run(), ref)


def test_shared_prefix_attention_of_hundreds_of_groups(cuda_device):
    # more rows and groups than the plan takes in one pass
    sizes = [2, 1, 3] * 100
    prefix = [64 + 5 * (g % 40) for g in range(300)]
    lens = [prefix[g] + (7 * r + g) % 90 for g, n in enumerate(sizes) for r in range(n)]
    for hd, block in ((32, 16), (128, 32)):
        b = Batch(cuda_device, sizes, prefix, lens, 4, 2, hd, block)
        b.check(b.run())


def test_shared_prefix_attention_repeats_and_keeps_its_inputs(cuda_device):
    b = Batch(cuda_device, [16, 8], [700, 300], [701 + i for i in range(16)] + [301 + 40 * i for i in range(8)], 32, 8,
              128, 256)
    kc, vc = b.kc.clone(), b.vc.clone()
    plan = shared_prefix_plan(b.lens, b.starts, b.prefix, 32, 8, 128, 256, b.tables.shape[1])
    out = b.run()
    for _ in range(3):
        assert torch.equal(b.run(plan=plan), out)  # one plan for every layer, the same bits every time
    assert torch.equal(b.kc.view(torch.int16), kc.view(torch.int16))
    assert torch.equal(b.vc.view(torch.int16), vc.view(torch.int16))
    b.check(out)


def test_shared_prefix_attention_refuses(cuda_device):
    b = Batch(cuda_device, [2], [64], [70, 80], 8, 2, 128, 16)
    plan = shared_prefix_plan(b.lens, b.starts, b.prefix, 8, 2, 128, 16, b.tables.shape[1])
    with pytest.raises(ValueError):  # a plan of another batch
        b.run(plan=plan._replace(rows=3))
    with pytest.raises(RuntimeError):
        b.run(plan=plan._replace(buf=plan.buf[:-1]))
    with pytest.raises(RuntimeError):
        shared_prefix_decode_attention(b.q.float(), b.kc, b.vc, b.tables, b.lens, b.starts, b.prefix)
    with pytest.raises(RuntimeError):
        shared_prefix_decode_attention(b.q, b.kc.half(), b.vc.half(), b.tables, b.lens, b.starts, b.prefix)
    with pytest.raises(RuntimeError):  # 16 dims a head
        shared_prefix_decode_attention(b.q[..., :16], b.kc[..., :16].contiguous(), b.vc[..., :16].contiguous(),
                                       b.tables, b.lens, b.starts, b.prefix)
    with pytest.raises(RuntimeError):  # a strided cache
        shared_prefix_decode_attention(b.q[..., :64], b.kc[..., :64], b.vc[..., :64], b.tables, b.lens, b.starts,
                                       b.prefix)
    with pytest.raises(ValueError):
        shared_prefix_decode_attention(b.q, b.kc, b.vc, b.tables, b.lens.cpu(), b.starts, b.prefix)
    with pytest.raises(RuntimeError):
        shared_prefix_decode_attention(b.q, b.kc.cpu(), b.vc, b.tables, b.lens, b.starts, b.prefix)
    b.check(b.run())


def test_refusals_with_numbers_raise(cuda_device):
    # a number in a message of the native library
    from rl_b200.ops.attention import paged_decode_attention
    from rl_b200.ops.norm import rms_norm

    b = Batch(cuda_device, [2], [64], [70, 80], 6, 2, 128, 16)
    with pytest.raises(RuntimeError, match="group size 3"):
        paged_decode_attention(b.q, b.kc, b.vc, b.tables, b.lens)
    with pytest.raises(RuntimeError, match="head_dim 24"):
        paged_decode_attention(b.q[:, :2, :24].contiguous(), b.kc[..., :24].contiguous(), b.vc[..., :24].contiguous(),
                               b.tables, b.lens)
    with pytest.raises(RuntimeError, match="unsupported dtype"), torch.no_grad():
        rms_norm(torch.zeros(2, 64, device=cuda_device, dtype=torch.float64),
                 torch.ones(64, device=cuda_device, dtype=torch.float64))


def test_shared_prefix_attention_reports_bad_device_data(cuda_device):
    from rl_b200.ops._ext import DeviceWaitError, check_device_errors

    check_device_errors()
    b = Batch(cuda_device, [2], [64], [70, 80], 8, 2, 128, 16)
    good = b.tables.clone()
    for bad in (b.kc.shape[0], -1, 2 ** 31 - 1):  # pages outside the cache are not read
        b.tables = good.clone()
        b.tables[1, 4] = bad
        b.run()
        with pytest.raises(DeviceWaitError, match="shared_prefix"):
            check_device_errors()
    b.tables = good
    for n in (16 * good.shape[1] + 9, 2 ** 31 - 1):  # longer than its table: cut there
        b.lens[1] = n
        b.run()
        with pytest.raises(DeviceWaitError, match="shared_prefix"):
            check_device_errors()
    b.lens[1] = 80
    b.starts = torch.tensor([2, 0], dtype=torch.int32, device=cuda_device)
    b.run()
    with pytest.raises(DeviceWaitError, match="shared_prefix"):
        check_device_errors()
    b.starts = torch.tensor([0, 2], dtype=torch.int32, device=cuda_device)
    b.check(b.run())


def test_shared_prefix_attention_scores_out_of_range(cuda_device):
    # a tile's first key is the reference of its scores: keys that exceed it by 2^15 and 2^60 (scores of up to
    # thousands), a first key whose score is -inf, late keys that outgrow everything before
    for fp8 in (False, True):
        b = Batch(cuda_device, [3], [600], [700, 610, 1500], 8, 2, 128, 16, fp8=fp8, q_scale=8.0)
        q = b.q[:, :1].clone()
        b.q = q.expand(-1, 8, -1).contiguous()
        t = b.tables.long()
        for row, page, slot, size in ((0, 0, 0, -30.0), (0, 20, 3, 25.0), (2, 60, 1, 45.0), (2, 90, 15, 90.0)):
            k = torch.sign(q[row, 0].float()) * size
            k = (k / b.k_scale).clamp(-448, 448) if fp8 else k
            b.kc[t[row, page], slot] = k.to(b.kc.dtype)
            if page < 37:
                for other in range(3):  # the prefix stays the same for every row
                    b.kc[t[other, page], slot] = k.to(b.kc.dtype)
        b.check(b.run())
    b = Batch(cuda_device, [3], [600], [700, 610, 1500], 8, 2, 128, 16)
    b.q = b.q.abs()
    b.kc[b.tables[0, 0].long(), 0] = float("-inf")  # of weight 0 for every query
    clean = b.run()
    assert torch.isfinite(clean).all()
    ref, tol = b.exact()
    assert ((clean.double() - ref).abs() <= tol.nan_to_num(nan=float("inf"))).all()


def test_shared_prefix_attention_many_rows_and_groups(cuda_device):
    g = torch.Generator().manual_seed(3)
    groups = torch.randint(0, 9, (150,), generator=g).tolist()
    prefix = torch.randint(0, 400, (150,), generator=g).tolist()
    lens = [max(1, p + int(x)) for n, p in zip(groups, prefix) for x in torch.randint(-20, 100, (n,), generator=g)]
    b = Batch(cuda_device, groups, prefix, lens, 4, 1, 64, 16, seed=5)
    b.check(b.run())


def test_shared_prefix_attention_far_pages(cuda_device):
    # pages behind 2^31 elements of the cache
    b = Batch(cuda_device, [3], [100], [130, 120, 300], 8, 8, 128, 256, pages=8400)
    assert int(b.tables.min()) * 256 * 8 * 128 > 2 ** 31
    b.check(b.run())


def test_shared_prefix_attention_streams_and_graphs(cuda_device):
    b = Batch(cuda_device, [4], [128], [140, 200, 150, 131], 8, 2, 128, 16, seed=1)
    c = Batch(cuda_device, [2, 2], [64, 300], [140, 100, 350, 331], 8, 2, 128, 16, seed=2)
    rb, rc = b.run(), c.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [b.run() for _ in range(20)]
    other = [c.run() for _ in range(20)]  # at the same time on the current stream
    s.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(o, rb) for o in outs) and all(torch.equal(o, rc) for o in other)
    graphs = []
    for x in (b, c):
        x.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = x.run()
        graphs.append((g, o))
    for _ in range(3):
        for g, _o in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], rb) and torch.equal(graphs[1][1], rc)
    # replayed on other lengths, groups and queries: planned again inside the graph
    b.lens.copy_(torch.tensor([64, 0, 150, 10], dtype=torch.int32))
    b.starts.copy_(torch.tensor([1, 4], dtype=torch.int32))
    b.q.mul_(0.5)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], b.run())
    b.check(graphs[0][1])


# ------------------------------------------------------------------- cache-page copies
@pytest.mark.parametrize("dtype,planes,block,nkv,hd", [
    (torch.bfloat16, (3, 2), 16, 2, 64), (torch.float8_e4m3fn, (2, 2), 256, 8, 128), (torch.float32, (1,), 5, 3, 7),
    (torch.float8_e4m3fn, (2,), 3, 1, 5), (torch.bfloat16, (2, 2), 64, 1, 4), (torch.bfloat16, (1, 2), 256, 8, 128)])
def test_copy_cache_pages(cuda_device, dtype, planes, block, nkv, hd):
    g = torch.Generator(device=cuda_device).manual_seed(0)
    pages = 40
    cache = torch.randn(*planes, pages, block, nkv, hd, device=cuda_device, generator=g).to(dtype)
    raw = cache.view(torch.uint8)
    want = raw.clone()
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    src = [order[i % 4] for i in range(30)]
    dst = order[4:34]
    tokens = [(7 * i) % (block + 1) for i in range(30)]
    for s, d, t in zip(src, dst, tokens):
        want[..., d, :t, :, :] = want[..., s, :t, :, :]
    copy_cache_pages(cache, src, dst, tokens)
    assert torch.equal(raw, want)
    want[..., order[39], :, :, :] = want[..., order[0], :, :, :]
    copy_cache_pages(cache, [order[0]], [order[39]])
    assert torch.equal(raw, want)


def test_copy_cache_pages_many_pairs(cuda_device):
    cache = torch.arange(2 * 4000 * 2 * 8, device=cuda_device, dtype=torch.int32).float().view(2, 4000, 2, 1, 8)
    want = cache.clone()
    src, dst = [i % 7 for i in range(3000)], list(range(1000, 4000))
    want[:, dst] = want[:, src]
    copy_cache_pages(cache, torch.tensor(src), torch.tensor(dst))
    assert torch.equal(cache, want)


def test_copy_cache_pages_views_and_odd_addresses(cuda_device):
    flat = torch.randn(4 * 6 * 8 * 2 * 8 + 3, device=cuda_device).bfloat16()
    cache = flat[3:].view(2, 2, 6, 8, 2, 8)  # not 16-byte aligned
    want = cache.clone()
    want[:, :, 4, :5] = want[:, :, 1, :5]
    copy_cache_pages(cache, [1], [4], [5])
    assert torch.equal(cache, want)
    assert torch.equal(cache, flat[3:].view_as(cache))


def test_copy_cache_pages_far_pages(cuda_device):
    cache = torch.zeros(2, 9000, 256, 8, 128, device=cuda_device, dtype=torch.bfloat16)  # 9.4 GB
    cache[1, 8990] = torch.randn(256, 8, 128, device=cuda_device).bfloat16()
    copy_cache_pages(cache, [8990, 8990], [8999, 3], [256, 100])
    assert torch.equal(cache[1, 8999], cache[1, 8990]) and torch.equal(cache[1, 3, :100], cache[1, 8990, :100])
    assert not cache[1, 3, 100:].any() and not cache[0].any()


def test_copy_cache_pages_refuses(cuda_device):
    cache = torch.randn(2, 2, 7, 4, 2, 8, device=cuda_device)
    before = cache.clone()
    for src, dst, tokens, error in [([1], [7], None, IndexError), ([-1], [2], None, IndexError),
                                    ([1], [2], [5], ValueError), ([1], [2], [-1], ValueError),
                                    ([1, 3], [2, 2], None, ValueError), ([1, 2], [2, 3], None, ValueError),
                                    ([1], [1], None, ValueError), ([2 ** 40], [1], None, IndexError),
                                    (torch.tensor([1], device=cuda_device), [2], None, ValueError)]:
        with pytest.raises(error):
            copy_cache_pages(cache, src, dst, tokens)
    with pytest.raises(TypeError):
        copy_cache_pages(cache, [1.5], [2])
    assert torch.equal(cache, before)


def test_copy_cache_pages_in_a_graph_and_on_a_stream(cuda_device):
    cache = torch.randn(2, 2, 7, 4, 2, 8, device=cuda_device)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        copy_cache_pages(cache, [0], [1])
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(g):
        copy_cache_pages(cache, [1, 1], [4, 5])
    cache[:, :, 1] = 7.0
    g.replay()
    torch.cuda.synchronize()
    assert (cache[:, :, 4] == 7).all() and (cache[:, :, 5] == 7).all() and not (cache[:, :, 6] == 7).any()


# ------------------------------------------------------------------------ norm with fp8 output
def _unfused(x, d, w, eps, mx):
    from rl_b200.ops.fp8_gemm import quant_act_mx
    from rl_b200.ops.norm import add_rms_norm, rms_norm
    from rl_b200.ops.quant import quant_fp8_group

    h, s = (rms_norm(x, w, eps), None) if d is None else add_rms_norm(x, d, w, eps)
    q, sc = quant_act_mx(h) if mx else quant_fp8_group(h, 128, False)
    return q, sc, s


@pytest.mark.parametrize("mx", [True, False])
@pytest.mark.parametrize("rows,H", [(1, 128), (1, 4096), (3, 384), (64, 4096), (129, 1536), (591, 5120), (592, 5120),
                                    (700, 128), (1000, 8192), (65, 8192), (600, 2048)])
@torch.no_grad()
def test_norm_fp8_equals_norm_then_quantisation(cuda_device, rows, H, mx):
    g = torch.Generator(device=cuda_device).manual_seed(rows + H)
    x, d = (torch.randn(rows, H, device=cuda_device, generator=g).bfloat16() for _ in range(2))
    x[0, :128] = 0  # a group of zeros
    d[0, :128] = 0
    w = (1 + 0.1 * torch.randn(H, device=cuda_device, generator=g)).bfloat16()
    for delta in (None, d):
        q, sc, s = _unfused(x, delta, w, 1e-5, mx)
        got = add_rms_norm_fp8(x, d, w, 1e-5, mx=mx) if delta is not None else rms_norm_fp8(x, w, 1e-5, mx=mx) + (None,)
        assert torch.equal(got[0].view(torch.uint8), q.view(torch.uint8))
        assert got[1].shape == sc.shape and torch.equal(got[1], sc)
        assert s is None or torch.equal(got[2], s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,H", [(2, 16384), (700, 256), (5, 640)])
@torch.no_grad()
def test_norm_fp8_against_64_bits(cuda_device, dtype, rows, H):
    g = torch.Generator(device=cuda_device).manual_seed(H)
    x, d = (torch.randn(rows, H, device=cuda_device, generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, device=cuda_device, generator=g)).to(dtype)
    half = torch.finfo(dtype).eps / 2
    for mx in (True, False):
        q, sc, s = add_rms_norm_fp8(x, d, w, 1e-5, mx=mx)
        total = x.double() + d.double()
        assert ((s.double() - total).abs() <= half * total.abs()).all()
        t = s.double()
        y = t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        sc = (sc[:, :rows].t() if mx else sc).double()
        got = (q.double().view(rows, -1, 128) * sc[..., None]).view(rows, H)
        # y is rounded to the input's type, then to e4m3: half a step of each (relative), below the normal
        # numbers half of e4m3's smallest step, 2^-10 of the scale; fp32 sums of H squares add H * 2^-24
        tol = y.abs() * (half + 2.0 ** -4 + H * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -10 * sc.repeat_interleave(128, 1)
        assert ((got - y).abs() <= tol).all()
        amax = y.view(rows, -1, 128).abs().amax(-1)
        slack = half + H * 2.0 ** -24 + 2.0 ** -20
        if mx:  # the smallest power of two that holds the group
            assert (torch.frexp(sc)[0] == 0.5).all()
            assert (sc * 448 >= amax * (1 - slack)).all() and (sc * 224 < amax * (1 + slack)).all()
        else:
            assert ((sc * 448 - amax).abs() <= slack * amax).all()


@torch.no_grad()
def test_norm_fp8_equals_norm_then_quantisation_for_every_exponent(cuda_device):
    # random mantissas and signs; x and delta of a row have exponents of a window of 16 (the first: subnormal
    # numbers and those next to them), or of all of them, so that most sums are inexact
    g = torch.Generator().manual_seed(3)
    rows = 16
    lo = torch.arange(rows)[:, None] * 16
    lo[-1] = 0
    width = torch.full((rows, 1), 16.0)
    width[-1] = 250.0

    def patterns():
        e = (lo + (torch.rand(rows, 512, generator=g) * width).long()).clamp(max=250)
        bits = (torch.randint(0, 2, e.shape, generator=g) << 15) | (e << 7) | torch.randint(0, 128, e.shape, generator=g)
        return (bits - ((bits >> 15) << 16)).to(torch.int16).view(torch.bfloat16).to(cuda_device)

    x, d = patterns(), patterns()
    w = (1 + 0.1 * torch.randn(512, generator=g)).bfloat16().to(cuda_device)
    for mx in (True, False):
        for eps in (1e-5, 1e-30):
            q, sc, s = _unfused(x, d, w, eps, mx)
            got = add_rms_norm_fp8(x, d, w, eps, mx=mx)
            assert torch.equal(got[2].view(torch.int16), s.view(torch.int16))
            assert torch.equal(got[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(got[1], sc)


@torch.no_grad()
def test_norm_fp8_special_values_views_and_empty(cuda_device):
    w = torch.ones(256, device=cuda_device).bfloat16()
    x = torch.randn(4, 256, device=cuda_device).bfloat16()
    x[1, 3] = float("nan")
    x[2] = 0
    for mx in (True, False):
        q, sc = rms_norm_fp8(x, w, mx=mx)
        assert q[1].float().isnan().all() and not q[2].float().any() and q[0].float().isfinite().all()
        assert torch.equal(q[3].view(torch.uint8), rms_norm_fp8(x[3:], w, mx=mx)[0][0].view(torch.uint8))
        q0, s0 = rms_norm_fp8(x[:0], w, mx=mx)
        assert q0.shape == (0, 256) and s0.shape == ((2, 128) if mx else (0, 2)) and (s0 == 1).all()
        flat = torch.cat([w[:1], x.flatten()])[1:]  # an odd address
        q1, sc1 = rms_norm_fp8(flat.view(4, 256), w, mx=mx)
        q2, sc2 = rms_norm_fp8(torch.cat([x, x], 1)[:, :256].view(2, 2, 256), w, mx=mx)  # strided rows
        for a, b in ((q1, sc1), (q2.view(4, 256), sc2)):
            assert torch.equal(a.view(torch.uint8), q.view(torch.uint8)) and torch.equal(b, sc)
    with pytest.raises(RuntimeError):
        rms_norm_fp8(torch.zeros(2, 16512, device=cuda_device), torch.ones(16512, device=cuda_device))
    with pytest.raises(ValueError):
        rms_norm_fp8(x, w.cpu())
    with pytest.raises(ValueError):
        rms_norm_fp8(x.double(), w.double())


# -------------------------------------------------------------------- the three together
def test_forked_pages_attend_like_copied_ones(cuda_device):
    # a prompt of 150 tokens in row 0's pages: forked (full pages shared, the last one copied) and copied whole
    b = Batch(cuda_device, [4], [150], [151, 180, 150, 200], 8, 2, 128, 16, share=False)
    want = b.run()
    b.check(want)
    storage = torch.stack([b.kc, b.vc])[None]  # [layers, 2, pages, block, heads, dims]
    own = b.tables.cpu()
    for forked in (True, False):
        cache, tables = storage.clone(), own.clone()
        first = 150 // 16 if forked else 0
        for r in range(1, 4):
            cache[0, :, own[r, :9].long()] = float("nan")  # the prompt's pages of the row, but the partly filled one's rest
            cache[0, :, own[r, 9].long(), :6] = float("nan")
            tables[r, :first] = own[0, :first]
        pairs = [(int(own[0, j]), int(own[r, j]), min(16, 150 - 16 * j)) for r in range(1, 4) for j in range(first, 10)]
        copy_cache_pages(cache, *zip(*pairs))
        b.kc, b.vc, b.tables = cache[0, 0], cache[0, 1], tables.to(cuda_device)
        assert torch.equal(b.run(), want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("graphs", [False, True])
def test_shared_prompt_rollout(cuda_device, graphs, fp8):
    """Prefill once, fork, decode with the shared prompt (and, fp8, with norms that quantise): the
    sampler's log-probs are the trainer's, within what rollouts with copied prompts are held to."""
    from rl_b200.distributed.batched_data_dict import BatchedDataDict
    from rl_b200.models.config import ModelConfig
    from rl_b200.models.policy.worker import PolicyWorker
    from rl_b200.parallel.state import single_process_state

    cfg = ModelConfig(name="small", vocab_size=2048, hidden_size=512, num_layers=3, num_heads=8, num_kv_heads=2,
                      head_dim=64, ffn_hidden_size=1408, rope_theta=10000.0, max_position_embeddings=1024)
    pcfg = {"model_name": "small", "max_total_sequence_length": 320, "precision": "bfloat16",
            "train_global_batch_size": 16, "train_micro_batch_size": 4,
            "generation": {"temperature": 1.0, "top_p": 1.0, "top_k": None, "max_new_tokens": 40,
                           "mcore_generation_config": {"block_size_tokens": 16,
                                                       "enable_shared_prefix_attention": True}},
            "sequence_packing": {"train_mb_tokens": 2048, "logprob_mb_tokens": 2048}}
    if fp8:
        pcfg["generation"]["vllm_cfg"] = {"precision": "fp8", "pow2_weight_scaling_factors": True,
                                          "pow2_activation_scaling_factors": True}
    w = PolicyWorker(pcfg, model_cfg=cfg, pstate=single_process_state(cuda_device), seed=0)
    assert w.engine.device.type == "cuda"
    w.engine.use_cuda_graphs = graphs
    w.engine.sync_every = 8
    w.engine.shared_prefix_min_bytes = 0
    g = torch.Generator().manual_seed(1)
    lens = torch.tensor([200, 33, 64, 257]).repeat_interleave(4)
    ids = torch.randint(0, 2048, (4, 257), generator=g).repeat_interleave(4, 0)
    data = BatchedDataDict({"input_ids": ids, "input_lengths": lens})
    try:
        for _ in range(2):  # the second call replays the first one's graphs
            out = w.generate(data)
            batch = BatchedDataDict({"input_ids": out["output_ids"],
                                     "input_lengths": out["unpadded_sequence_lengths"]})
            lp = w.get_logprobs(batch)["logprobs"]
            mask = torch.zeros_like(lp, dtype=torch.bool)
            for i in range(16):
                mask[i, int(lens[i]): int(out["unpadded_sequence_lengths"][i])] = True
            diff = (lp - out["logprobs"])[mask].abs()
            assert mask.sum() > 16 and float(diff.mean()) < (0.1 if fp8 else 0.02)
            _ext.check_device_errors()
            assert w.engine._prompts is not None
        # a prompt too short to pay is forked, and attended to row by row
        w.engine.shared_prefix_min_bytes = 1 << 40
        out = w.generate(data)
        assert w.engine._prompts is None
        lp = w.get_logprobs(BatchedDataDict({"input_ids": out["output_ids"],
                                             "input_lengths": out["unpadded_sequence_lengths"]}))["logprobs"]
        mask = torch.zeros_like(lp, dtype=torch.bool)
        for i in range(16):
            mask[i, int(lens[i]): int(out["unpadded_sequence_lengths"][i])] = True
        assert float((lp - out["logprobs"])[mask].abs().mean()) < (0.1 if fp8 else 0.02)
    finally:
        w.shutdown()
    assert w.engine.stats_last_prefill["prefilled"] == 4


# ------------------------------------------------------- long tails, far scores, other head counts
@pytest.mark.parametrize("binades", [20.5, 25.5, 27.5])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 4, 64), (32, 8, 128)])
def test_shared_prefix_attention_fp8_long_tail(cuda_device, nq, nkv, hd, binades):
    # one key of large score whose value is 0, and a thousand whose weights are 2^-binades of its: they alone make
    # the output.  f16 weights are normal numbers down to 2^-28 of the largest (half a step: the bound's 2^-11).
    lens = [1024 + 7 * i for i in range(40)] + [1500] * 16
    b = Batch(cuda_device, [16], [1472], lens, nq, nkv, hd, 64, fp8=True, alone=(40, 0))
    live = b.kc.float().isfinite()
    b.q.fill_(1.0)
    b.kc.copy_(torch.where(live, 0.0, b.kc.float()).to(b.kc.dtype))
    b.vc.copy_(torch.where(live, b.vc.float().abs().clamp(min=1.0), b.vc.float()).to(b.vc.dtype))
    first = b.tables[:, 0].long()
    b.kc[first, 0] = torch.tensor(4.0, device=cuda_device).to(b.kc.dtype)
    b.vc[first, 0] = torch.tensor(0.0, device=cuda_device).to(b.vc.dtype)
    scale = binades * math.log(2) / (4.0 * b.k_scale * hd)
    b.check(b.run(scale=scale), scale=scale)


@pytest.mark.parametrize("size", [2.0 ** 19, 2.0 ** 21, 2.0 ** 25, 2.0 ** 26, 2.0 ** 40, -2.0 ** 19, -2.0 ** 26])
def test_shared_prefix_attention_fp8_scores_of_millions(cuda_device, size):
    # every key scores the same +-size (in powers of two), so every weight is the same number exactly: sums and the
    # output's rounding are all that is off; then one shared key scores the opposite and is all or nothing
    b = Batch(cuda_device, [2], [300], [310, 700], 8, 2, 128, 16, fp8=True)
    b.q.fill_(1.0)
    live = b.kc.float().isfinite()
    scale = size * math.log(2) / (128 * b.k_scale)
    b.kc.copy_(torch.where(live, 1.0, b.kc.float()).to(b.kc.dtype))
    page, slot = int(b.tables[0, 12]), 8  # key 200
    for opposite in (False, True):
        if opposite:
            b.kc[page, slot] = torch.tensor(-1.0, device=cuda_device).to(b.kc.dtype)
        got = b.run(scale=scale)
        for r, n in enumerate((310, 700)):
            t = torch.arange(n, device=cuda_device)
            slots = b.tables[r].long()[t // 16] * 16 + t % 16
            v = b.vc.view(-1, 2, 128)[slots].double() * b.v_scale
            if opposite:
                v = v[200:201] if size < 0 else torch.cat([v[:200], v[201:]])
            want = v.mean(0).repeat_interleave(4, 0)
            tol = n * 2.0 ** -23 * v.abs().mean(0).repeat_interleave(4, 0) + 2.0 ** -8 * want.abs() + 1e-30
            assert ((got[r].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("size", [2.0 ** 23, 2.0 ** 26, 2.0 ** 31, 2.0 ** 40, 1e32, -2.0 ** 26, -2.0 ** 40, -1e32])
def test_shared_prefix_attention_equal_scores_of_any_size(cuda_device, hd, size):
    # every key scores the same, so every weight is 1 exactly, whatever the scores' size: sums, P's type and the
    # output's rounding are all that is off; then one shared key scores the opposite and is all or nothing
    b = Batch(cuda_device, [3], [400], [410, 700, 1500], 8, 2, hd, 16)
    b.q.fill_(1.25)
    live = b.kc.float().isfinite()
    b.kc.copy_(torch.where(live, 1.0, b.kc.float()).to(b.kc.dtype))
    page, slot = int(b.tables[0, 12]), 8  # key 200
    for opposite in (False, True):
        if opposite:
            b.kc[page, slot] = -1.0
        got = b.run(scale=size / (1.25 * hd))
        for r, n in enumerate((410, 700, 1500)):
            t = torch.arange(n, device=cuda_device)
            slots = b.tables[r].long()[t // 16] * 16 + t % 16
            v = b.vc.view(-1, 2, hd)[slots].double()
            if opposite:
                v = v[200:201] if size < 0 else torch.cat([v[:200], v[201:]])
            want = v.mean(0).repeat_interleave(4, 0)
            tol = n * 2.0 ** -23 * v.abs().mean(0).repeat_interleave(4, 0) + 2.0 ** -8 * want.abs() + 1e-30
            assert ((got[r].double() - want).abs() <= tol).all()


def test_shared_prefix_attention_scores_far_below_zero(cuda_device):
    # a first key of -inf (the reference of the tiles' scores), then scores of -1e32 and less: the second key's value
    # is the output, next to it no weight is above 0
    for hd in (64, 128):
        b = Batch(cuda_device, [2], [300], [310, 700], 8, 2, hd, 16)
        b.q.fill_(1e16)
        for r, n in enumerate([310, 700]):
            t = torch.arange(n, device=cuda_device)
            k = -1e14 * (1 + t.double())
            k[0] = float("-inf")
            slot = b.tables[r].long()[t // 16] * 16 + t % 16
            b.kc.view(-1, 2, hd)[slot] = k.to(torch.bfloat16)[:, None, None].expand(-1, 2, hd)
        out = b.run()
        v = b.vc[b.tables[:, 0].long(), 1]
        assert torch.equal(out.view(2, 2, 4, hd), v[:, :, None].expand(-1, -1, 4, -1))


@pytest.mark.parametrize("hd", [64, 128])
def test_shared_prefix_attention_first_key_of_weight_zero(cuda_device, hd):
    # as in test_shared_prefix_attention_scores_out_of_range, with the bound of the keys that count: over all of them
    # it is infinite (the sum of |q k| is)
    b = Batch(cuda_device, [3], [600], [700, 610, 1500], 8, 2, hd, 16)
    b.q = b.q.abs().clamp(min=2.0 ** -6)
    b.kc[b.tables[0, 0].long(), 0] = float("-inf")
    got = b.run()
    for r, n in enumerate(b.lens.tolist()):  # the row by itself behind its first key, in pages of one key
        t = torch.arange(1, n, device=cuda_device)
        row = object.__new__(Batch)
        row.__dict__.update(b.__dict__, bs=1, q=b.q[r:r + 1], lens=b.lens[r:r + 1] - 1,
                            tables=(b.tables[r].long()[t // 16] * 16 + t % 16)[None])
        ref, tol = row.exact()
        assert torch.isfinite(ref).all() and float(tol.max()) < 0.25
        assert ((got[r:r + 1].double() - ref).abs() <= tol).all()


def _rollout_worker(dev, heads, kv_heads, head_dim, vocab=2048, stop=(), vllm=None, layers=2):
    from rl_b200.models.config import ModelConfig
    from rl_b200.models.policy.worker import PolicyWorker
    from rl_b200.parallel.state import single_process_state

    cfg = ModelConfig(name="small", vocab_size=vocab, hidden_size=512, num_layers=layers, num_heads=heads,
                      num_kv_heads=kv_heads, head_dim=head_dim, ffn_hidden_size=1408, rope_theta=10000.0,
                      max_position_embeddings=1024)
    pcfg = {"model_name": "small", "max_total_sequence_length": 320, "precision": "bfloat16",
            "train_global_batch_size": 16, "train_micro_batch_size": 4,
            "generation": {"temperature": 1.0, "top_p": 1.0, "top_k": None, "max_new_tokens": 40,
                           "stop_token_ids": list(stop), "vllm_cfg": vllm or {},
                           "mcore_generation_config": {"block_size_tokens": 16,
                                                       "enable_shared_prefix_attention": True}},
            "sequence_packing": {"train_mb_tokens": 2048, "logprob_mb_tokens": 2048}}
    return PolicyWorker(pcfg, model_cfg=cfg, pstate=single_process_state(dev), seed=0), cfg


def _rollout_batch(copies, vocab=2048):
    from rl_b200.distributed.batched_data_dict import BatchedDataDict

    g = torch.Generator().manual_seed(1)
    n = 16 // copies
    lens = torch.tensor(([200, 33, 64, 257] * 4)[:n]).repeat_interleave(copies)
    ids = torch.randint(0, vocab, (n, 257), generator=g).repeat_interleave(copies, 0)
    return BatchedDataDict({"input_ids": ids, "input_lengths": lens})


def _logprob_gap(w, data, out):
    from rl_b200.distributed.batched_data_dict import BatchedDataDict

    lp = w.get_logprobs(BatchedDataDict({"input_ids": out["output_ids"],
                                         "input_lengths": out["unpadded_sequence_lengths"]}))["logprobs"]
    mask = torch.zeros_like(lp, dtype=torch.bool)
    for i, n in enumerate(data["input_lengths"].tolist()):
        mask[i, n: int(out["unpadded_sequence_lengths"][i])] = True
    return float((lp - out["logprobs"])[mask].abs().mean())


@pytest.mark.parametrize("spec", [False, True])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
@pytest.mark.parametrize("copies", [4, 1])
@pytest.mark.parametrize("heads,head_dim", [(14, 128), (6, 64)])
def test_rollout_of_heads_that_only_shared_prompts_take(cuda_device, heads, head_dim, copies, kv, spec, monkeypatch):
    # query heads per KV head that row-by-row attention lacks: prompts too short to pay, with copies and without
    import dataclasses

    from rl_b200.models.transformer import TransformerLM

    w, cfg = _rollout_worker(cuda_device, heads, 2, head_dim, vllm={"kv_cache_dtype": kv})
    w.engine.sync_every = 8
    if spec:
        w.engine.set_draft(TransformerLM(dataclasses.replace(cfg, num_layers=1), device=cuda_device,
                                         dtype=torch.bfloat16, seed=9), 3)
    data = _rollout_batch(copies)
    try:
        out = w.generate(data)
        assert _logprob_gap(w, data, out) < (0.1 if kv == "fp8" else 0.02)
        _ext.check_device_errors()
        if heads == 6 and copies == 1:  # more rows than a plan takes: refused before the prefill
            monkeypatch.setattr("rl_b200.models.generation.engine._PLAN_ROWS", 63 if spec else 15)
            with pytest.raises(ValueError, match="16 sequences"):
                w.generate(data)
    finally:
        w.shutdown()


@pytest.mark.parametrize("heads", [8, 6])
def test_rollout_decides_again_for_the_rows_that_are_left(cuda_device, heads):
    # 16 rows save 851 kB a layer, the 8 rows or fewer of the next batch 702 kB at most (4 of 257 and 4 of 200 tokens)
    w, _ = _rollout_worker(cuda_device, heads, 2, 64, vocab=256, stop=range(8))
    w.engine.sync_every = 8
    w.engine.shared_prefix_min_bytes = 750_000
    seen, state = [], w.engine._state
    w.engine._state = lambda nb, max_new, key: (seen.append((nb, key[-1])), state(nb, max_new, key))[1]
    data = _rollout_batch(4, 256)
    try:
        out = w.generate(data)
        assert seen[0] == (16, True) and len(seen) > 1 and seen[1][0] <= 8
        # 3 query heads per KV head have no other way
        assert all(shares == (heads == 6) for _, shares in seen[1:])
        assert _logprob_gap(w, data, out) < 0.02
        _ext.check_device_errors()
    finally:
        w.shutdown()


def test_copy_cache_pages_launches(cuda_device):
    cache = torch.zeros(2, 1300, 2, 1, 8, device=cuda_device)
    for src, dst, tokens, launches in (([], [], None, 0), ([0], [1], [0], 0), ([0], [1], None, 1),
                                       ([0] * 641, list(range(1, 642)), None, 2)):
        before = _ext.launch_count()
        copy_cache_pages(cache, src, dst, tokens)
        assert _ext.launch_count() - before == launches
