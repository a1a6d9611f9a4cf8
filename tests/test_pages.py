"""The paged key/value store on the GPU: codes against the framework's own
codec, values read back, and attention against a plain evaluation in 64 bits.

Tolerances (from the number formats, before any run).  u is half the spacing of
the output type at 1: 2^-8 (bf16), 2^-11 (f16).  With A = sum p|v| / sum p,
L = max over visible tokens of scale * sum_d |q_d k_d|:
  output rounding                                   u |o|
  softmax weights rounded to the operand type       u A   (bf16), 2^-11 A (codes: f16 operands)
  codes: dequantized values rounded to f16          2^-11 A
  codes: keys rounded to f16 move a logit by        2^-11 L, the weights and their sum alike: 2 * 2^-11 L A
  fp32 sums of products, exp2, scaling              2^-17 (1 + 2 L) A
A row's log-sum-exp moves by at most its logits' error.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import kivi_cache as K

    return torch, K


TYPES = {"bf16": "bfloat16", "f16": "float16", "f32": "float32"}
HALF = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}


class Case:
    """A store with its sequences: new[b] newest tokens of kv[b] (whose history
    the pool already holds), pages in random order, every byte that no sequence
    owns poisoned."""

    def __init__(self, env, new, kv, heads=2, group=4, dim=128, page=16, bits=16, kind="bf16", pool=None, seed=0,
                 spread=0.5):
        torch, K = env
        self.torch, self.K = torch, K
        self.new, self.kv, self.heads, self.group, self.dim, self.page, self.bits = new, kv, heads, group, dim, page, bits
        self.kind, self.dtype = kind, getattr(torch, TYPES[kind])
        pool = pool or ("bf16" if kind == "f32" else kind)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        used = [-(-n // page) for n in kv]
        self.pages = sum(used) + 2
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv), max(1, max(used)) + 1), -7, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.total, self.cu_host = int(cu[-1]), cu
        self.cu = torch.from_numpy(cu).cuda()
        self.kv_lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
        self.config = K.PagesConfig(bits=bits, dtype=pool, num_pages=self.pages, page_size=page, num_kv_heads=heads,
                                    head_dim=dim)
        self.params = [None, None]
        if bits == 16:
            nan = float("nan")
            self.data = [torch.full((self.pages, heads, page, dim), nan, dtype=getattr(torch, TYPES[pool]), device="cuda")
                         for _ in range(2)]
        else:
            self.data = [torch.full((self.pages, heads, page, dim * bits // 8), 255, dtype=torch.uint8, device="cuda")
                         for _ in range(2)]
            self.params = [torch.full((self.pages, heads, page, 2), float("nan"), device="cuda") for _ in range(2)]
        self.store = K.KvPages(self.config, *self.data, *self.params)
        gain = torch.exp(spread * torch.randn(heads, dim, generator=g, device="cuda"))
        # whole sequences go in first, as a batch whose newest tokens are all of them
        hcu = np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)
        whole = self.batch(self.torch.from_numpy(hcu).cuda(), int(hcu[-1]), max(max(kv), 1))
        self.k = (torch.randn(int(hcu[-1]), heads, dim, generator=g, device="cuda") * gain).to(self.dtype)
        self.v = torch.randn(int(hcu[-1]), heads, dim, generator=g, device="cuda").to(self.dtype)
        self.whole, self.hcu = whole, hcu
        self.store.write_dev(whole, self.k, self.v)
        self.step = self.batch(self.cu, self.total, max(max(new), 1))

    def batch(self, cu, total, most):
        return self.K.PagesBatch(self.table, cu, self.kv_lens, total, most)

    def held(self, side):
        """Every sequence's rows as the pool holds them, 64 bits, from its bytes."""
        torch = self.torch
        out = []
        for b, n in enumerate(self.kv):
            t = torch.arange(n, device="cuda")
            p = self.table[b].long()[t // self.page]
            x = self.data[side][p, :, t % self.page]
            if self.bits == 16:
                out.append(x.double())
                continue
            if self.bits == 4:
                x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
            q = self.params[side][p, :, t % self.page].double()
            out.append(q[..., 1:] + q[..., :1] * x.double())
        return out

    def queries(self, heads=None):
        torch = self.torch
        return torch.randn(self.total, self.heads * self.group, self.dim, generator=self.g, device="cuda").to(self.dtype)

    def attend(self, q, scale, window=0, sinks=0, lse=True, **kw):
        torch = self.torch
        out = torch.full_like(q, float("nan"))
        l = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None
        self.store.attention_dev(self.step, q, self.heads * self.group, scale, out, window=window, sinks=sinks, d_lse=l, **kw)
        torch.cuda.synchronize()
        self.store.status()
        return out, l

    def reference(self, q, scale, window=0, sinks=0):
        """(o, lse, tolerance of o, tolerance of lse) in 64 bits."""
        torch = self.torch
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(o)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        ltol = torch.zeros_like(lse)
        u = HALF[self.kind]
        uw = u if self.bits == 16 else 2.0**-11
        for b, (k, v) in enumerate(zip(self.held(0), self.held(1))):
            n, kv, s = self.new[b], self.kv[b], int(self.cu_host[b])
            t = torch.arange(kv, device="cuda")
            for i in range(n):
                p = kv - n + i
                see = t <= p
                if window:
                    see &= (t > p - window) | (t < sinks)
                if not bool(see.any()):
                    continue
                kk, vv = k[see], v[see]
                for h in range(self.heads):
                    qq = q[s + i, h * self.group:(h + 1) * self.group].double()
                    x = qq @ kk[:, h].T * scale
                    big = (qq.abs() @ kk[:, h].abs().T * abs(scale)).amax(-1)
                    w = torch.softmax(x, -1)
                    rows = slice(h * self.group, (h + 1) * self.group)
                    o[s + i, rows] = w @ vv[:, h]
                    a = w @ vv[:, h].abs()
                    move = big * (2.0**-11 if self.bits < 16 else 0.0) + 2.0**-17 * (1 + big)
                    rel = uw + (2.0**-11 if self.bits < 16 else 0.0) + 2 * move
                    tol[s + i, rows] = u * o[s + i, rows].abs() + a * rel[:, None] * (1 + u) + 2.0**-24
                    lse[s + i, rows] = torch.logsumexp(x, -1)
                    ltol[s + i, rows] = move + 2.0**-20 * (1 + lse[s + i, rows].abs())
        return o, lse, tol, ltol

    def check(self, q, scale, window=0, sinks=0):
        torch = self.torch
        out, lse = self.attend(q, scale, window, sinks)
        o, l, tol, ltol = self.reference(q, scale, window, sinks)
        d = (out.double() - o).abs()
        assert bool((d <= tol).all()), float((d / tol.clamp(min=1e-300)).nan_to_num(nan=math.inf).max())
        empty = torch.isinf(l)
        assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all())
        dl = (lse.double() - l)[~empty].abs()
        assert bool((dl <= ltol[~empty]).all()), float((dl / ltol[~empty]).max())
        return out, lse


# ------------------------------------------------------------------ writing and reading


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kind,dim,page,heads", [("f32", 128, 16, 3), ("bf16", 64, 64, 2), ("f16", 96, 32, 1),
                                                 ("bf16", 32, 256, 5)])
def test_codes_equal_the_per_token_codec(env, bits, kind, dim, page, heads):
    torch, K = env
    c = Case(env, [1, 1, 0], [37, 300, 0], heads=heads, group=1, dim=dim, page=page, bits=bits, kind=kind)
    for side, x in enumerate((c.k, c.v)):
        for b, n in enumerate(c.kv):
            if not n:
                continue
            rows = x[int(c.hcu[b]):int(c.hcu[b + 1])].float().cpu().numpy()  # [n, heads, dim]
            t = K.quantize_per_token(np.ascontiguousarray(rows.transpose(1, 0, 2)), 1, heads, n, dim, bits, dim)
            at = torch.arange(n, device="cuda")
            p = c.table[b].long()[at // page]
            codes = c.data[side][p, :, at % page].permute(1, 0, 2).contiguous().cpu().numpy()
            params = c.params[side][p, :, at % page].permute(1, 0, 2).contiguous().cpu().numpy()
            assert (codes.reshape(-1).view(np.uint32) == np.asarray(t.codes, np.uint32).reshape(-1)).all()
            assert (params.reshape(-1).view(np.uint32) == np.asarray(t.params, np.float32).reshape(-1).view(np.uint32)).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("kind,dim,page", [("f32", 64, 16), ("bf16", 128, 32), ("f16", 96, 128)])
def test_read_back(env, bits, kind, dim, page):
    """Whole sequences and the newest tokens alone come back as the bytes stand for."""
    torch, K = env
    c = Case(env, [1, 5, 40, 0], [1, 77, 40, 19], heads=3, dim=dim, page=page, bits=bits, kind=kind)
    held = [torch.cat(c.held(s)) for s in (0, 1)]
    for batch, pick in ((c.whole, None), (c.step, c.new)):
        k = torch.full((batch.total_tokens, 3, dim), float("nan"), dtype=c.dtype, device="cuda")
        v = torch.full_like(k, float("nan"))
        c.store.read_dev(batch, k, v)
        c.store.status()
        for got, want in zip((k, v), held):
            if pick is not None:
                want = torch.cat([want[int(c.hcu[b + 1]) - n:int(c.hcu[b + 1])] for b, n in enumerate(pick)])
            if bits == 16 and kind != "f32":
                assert torch.equal(got.double(), want)
            else:  # one fused multiply-add in fp32, then the output's rounding
                assert bool(((got.double() - want).abs() <= (HALF[kind] + 2.0**-22) * want.abs() + 2.0**-20).all())


def test_strided_and_unaligned_rows(env):
    """Keys and values as slices of one fused projection, and rows that start off
    16-byte boundaries, give the bytes of contiguous ones."""
    torch, K = env
    for off in (0, 1):
        c = Case(env, [3, 50], [9, 50], heads=2, bits=8, dim=64, page=16)
        want = [d.clone() for d in c.data + c.params]
        total = c.whole.total_tokens
        fused = torch.zeros(total, 7, 64 + off, dtype=c.dtype, device="cuda")
        fused[:, 2:4, off:] = c.k
        fused[:, 5:7, off:] = c.v
        for d in c.data + c.params:
            d.fill_(0)
        c.store.write_dev(c.whole, fused[:, 2:4, off:], fused[:, 5:7, off:])
        c.store.status()
        for b, n in enumerate(c.kv):
            t = torch.arange(n, device="cuda")
            p = c.table[b].long()[t // 16]
            for got, w in zip(c.data + c.params, want):
                assert torch.equal(got[p, :, t % 16], w[p, :, t % 16])
        back = torch.zeros(total, 7, 64 + off, dtype=c.dtype, device="cuda")
        c.store.read_dev(c.whole, back[:, 2:4, off:], back[:, 5:7, off:])
        k, v = torch.empty_like(c.k), torch.empty_like(c.v)
        c.store.read_dev(c.whole, k, v)
        assert torch.equal(back[:, 2:4, off:], k) and torch.equal(back[:, 5:7, off:], v)
        assert bool((back[:, :2] == 0).all()) and bool((back[:, 4] == 0).all())


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_write_touches_its_own_rows_alone(env, bits):
    torch, K = env
    c = Case(env, [3, 1, 2], [20, 33, 2], heads=2, bits=bits, dim=32, page=16)
    before = [d.clone() for d in c.data + [p for p in c.params if p is not None]]
    k = torch.randn(6, 2, 32, device="cuda").to(c.dtype)
    c.store.write_dev(c.step, k, -k)
    c.store.status()
    own = torch.zeros(c.pages, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.new):
        t = torch.arange(c.kv[b] - n, c.kv[b], device="cuda")
        own[c.table[b].long()[t // 16], t % 16] = True
    for d, w in zip(c.data + [p for p in c.params if p is not None], before):
        same = (d.view(torch.uint8) == w.view(torch.uint8)).all(-1)
        assert bool(same.permute(0, 2, 1)[~own].all())
        assert not bool(same.permute(0, 2, 1)[own].all())


def test_codes_of_constant_and_extreme_rows(env):
    torch, K = env
    c = Case(env, [4], [4], heads=1, bits=8, dim=32, page=16, kind="f32")
    x = torch.zeros(4, 1, 32, device="cuda")
    x[0] = 3.25                      # constant: scale 0
    x[1, 0, 0], x[1, 0, 1] = 1e30, -1e30
    x[2, 0, 5] = float("nan")        # code 0, skipped by the range
    x[2, 0, 6] = 2.0
    x[3] = torch.arange(32, device="cuda") * 1e-42  # subnormal span
    c.store.write_dev(c.step, x, x)
    k, v = torch.empty_like(x), torch.empty_like(x)
    c.store.read_dev(c.step, k, v)
    t = K.quantize_per_token(x.cpu().numpy().reshape(-1), 1, 1, 4, 32, 8, 32)
    at = torch.arange(4, device="cuda")
    codes = c.data[0][c.table[0].long()[at // 16], :, at % 16].contiguous().cpu().numpy().reshape(-1).view(np.uint32)
    assert (codes == np.asarray(t.codes, np.uint32).reshape(-1)).all()
    assert bool((k[0] == 3.25).all()) and torch.equal(k, v)


# ------------------------------------------------------------------ attention

DECODE = [
    dict(new=[1], kv=[1]),
    dict(new=[1, 1, 1], kv=[1, 16, 17], group=8),
    dict(new=[1] * 5, kv=[700, 3, 64, 65, 1000], group=1, heads=3, dim=64, page=64),
    dict(new=[1, 0, 1], kv=[300, 5, 129], group=7, dim=96, page=32),
    dict(new=[1] * 3, kv=[0, 900, 257], group=3, dim=32, page=256),
    dict(new=[1, 1], kv=[5000, 333], group=16, heads=1, page=128),
    dict(new=[1], kv=[20011], group=5, heads=1, page=16),
]
CHUNK = [
    dict(new=[2], kv=[2], group=1, heads=1),
    dict(new=[33], kv=[33], group=4),
    dict(new=[5, 1, 0, 128], kv=[300, 400, 9, 128], group=4, page=32),
    dict(new=[130, 7], kv=[513, 1000], group=8, heads=1, page=64),
    dict(new=[200], kv=[200], group=3, dim=64, page=128),
    dict(new=[64, 3], kv=[40, 2], group=2, dim=96, page=16),   # more new tokens than the cache counts: empty rows
    dict(new=[17, 300], kv=[2100, 400], group=1, dim=32, page=256, heads=3),
    dict(new=[4], kv=[9000], group=16, heads=1, page=64),
    dict(new=[6] * 9, kv=[150 * i + 6 for i in range(9)], group=5, heads=1, page=16),
    dict(new=[400], kv=[3777], group=4, page=64),
    dict(new=[90, 260], kv=[2600, 1311], group=6, heads=3, dim=64, page=16),
    dict(new=[1100], kv=[1100], group=1, heads=1, page=256),
    dict(new=[214, 61, 1], kv=[2601, 62, 1], group=33, heads=3, dim=96, page=32),  # short blocks after long ones
    dict(new=[2], kv=[0], group=33, heads=1, dim=64, page=256),
]
MASKS = [(1, 0), (1, 3), (17, 0), (64, 4), (100, 21), (128, 200), (5000, 4)]


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (16, "f16"), (8, "bf16"), (8, "f16"), (4, "bf16"), (4, "f16")])
@pytest.mark.parametrize("i", range(len(DECODE) + len(CHUNK)))
def test_attention(env, i, bits, kind):
    c = Case(env, bits=bits, kind=kind, seed=i, **(DECODE + CHUNK)[i])
    c.check(c.queries(), 1.0 / math.sqrt(c.dim))


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "f16"), (4, "bf16")])
@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("i", [2, 3, 6, 9, 10, 13, 16, 17, 18])
def test_window_and_first_tokens(env, i, window, sinks, bits, kind):
    c = Case(env, bits=bits, kind=kind, seed=50 + i, **(DECODE + CHUNK)[i])
    c.check(c.queries(), 1.0 / math.sqrt(c.dim), window, sinks)


@pytest.mark.parametrize("i", [2, 9, 10])
def test_hidden_pages_are_not_needed(env, i):
    """Pages that no row sees may have been freed: entries out of range, NaN inside."""
    torch, K = env
    c = Case(env, bits=16, **(DECODE + CHUNK)[i])
    window, sinks = 20, 3
    q = c.queries()
    want, wlse = c.attend(q, 0.1, window, sinks)
    for b, (n, kv) in enumerate(zip(c.new, c.kv)):
        for j in range(-(-kv // c.page)):
            lo, hi = j * c.page, min(kv, (j + 1) * c.page)
            if lo >= sinks and hi - 1 <= kv - n - window:
                c.data[0][c.table[b, j].long()] = float("nan")
                c.data[1][c.table[b, j].long()] = float("inf")
                c.table[b, j] = -1
    got, lse = c.attend(q, 0.1, window, sinks)
    assert torch.equal(got, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_unseen_infinities_and_nan_do_not_leak(env, bits, bad):
    """A newest token whose key and value are not finite reaches the rows that
    see it and no other row of its tile."""
    torch, K = env
    new, kv, at = 70, 200, 30  # row `at` of the chunk holds the bad token
    c = Case(env, [new], [kv], heads=1, group=4, bits=bits)
    q = c.queries()
    want, _ = c.attend(q, 0.1)
    x = torch.randn(new, 1, 128, device="cuda", generator=c.g).to(c.dtype)
    k, v = c.k[kv - new:].clone(), c.v[kv - new:].clone()
    v[at, 0, 5] = bad
    k[at, 0, 7] = bad
    c.store.write_dev(c.step, k, v)
    got, _ = c.attend(q, 0.1)
    assert torch.equal(got[:at], want[:at])
    assert bool((~torch.isfinite(got[at:, :, 5].float())).all()) or bits == 8
    # under a window the token is out of sight again for the last rows
    want, _ = c.attend(q, 0.1, 16, 2)
    assert bool(torch.isfinite(want[at + 16:].float()).all()) and bool(torch.isfinite(want[:at].float()).all())


@pytest.mark.parametrize("i", [5, 12])
@pytest.mark.parametrize("bits", [16, 4])
def test_large_logits_and_negative_scale(env, i, bits):
    """Weights concentrated on one token, references that move often."""
    c = Case(env, bits=bits, seed=7, spread=1.5, **(DECODE + CHUNK)[i])
    q = c.queries()
    q[:, 0] *= 8
    c.check(q, 0.3)
    c.check(q, -0.3)
    c.check(q, 0.0)


def test_strided_queries_and_outputs(env):
    torch, K = env
    for spec in (DECODE[2], CHUNK[2]):
        for off in (0, 1):
            c = Case(env, bits=16, **spec)
            hq, d = c.heads * c.group, c.dim
            q = c.queries()
            want, lse = c.attend(q, 0.1)
            big = torch.zeros(c.total, hq + 3, d + off, dtype=c.dtype, device="cuda")
            big[:, 2:2 + hq, off:] = q
            out = torch.zeros(hq + 1, c.total, d + off, dtype=c.dtype, device="cuda")
            view = out.permute(1, 0, 2)[:, :hq, off:]
            c.store.attention_dev(c.step, big[:, 2:2 + hq, off:], hq, 0.1, view)
            torch.cuda.synchronize()
            assert torch.equal(view, want)
            assert bool((out[hq] == 0).all())


@pytest.mark.parametrize("i", [2, 6, 9, 11, 14])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_same_bits_every_time(env, i, bits):
    torch, K = env
    c = Case(env, bits=bits, **(DECODE + CHUNK)[i])
    q = c.queries()
    a, la = c.attend(q, 0.1)
    for _ in range(3):
        b, lb = c.attend(q, 0.1)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_streams_and_graphs(env):
    """Calls on several streams share a handle's scratch safely, and a captured
    step follows the lengths that device memory holds when it replays."""
    torch, K = env
    c = Case(env, bits=16, **DECODE[6])
    q = c.queries()
    want, _ = c.attend(q, 0.1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty_like(q) for _ in range(12)]
    torch.cuda.synchronize()
    for j, o in enumerate(outs):
        c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, o, stream=streams[j % 3])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    s = torch.cuda.Stream()
    out = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, out, stream=s)
    for n in (20011, 1777, 40):
        c.kv_lens.fill_(n)
        ref, _ = c.attend(q, 0.1)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_an_offset_past_32_bits(env):
    """Rows beyond 2^31 bytes of the store, written, read and attended over."""
    torch, K = env
    pages, heads, page, dim = 70000, 4, 64, 128  # 4.6 GB a side
    data = [torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    store = K.KvPages(K.PagesConfig(num_pages=pages, page_size=page, num_kv_heads=heads), *data)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    n = 150
    k = torch.randn(n, heads, dim, device="cuda").bfloat16()
    v = torch.randn(n, heads, dim, device="cuda").bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    whole = K.PagesBatch(table, torch.tensor([0, n], dtype=torch.int32, device="cuda"), lens, n, n)
    store.write_dev(whole, k, v)
    assert torch.equal(data[0][pages - 1, :, 3], k[3])
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    store.read_dev(whole, kb, vb)
    assert torch.equal(kb, k) and torch.equal(vb, v)
    for m in (1, 20):
        q = torch.randn(m, heads, dim, device="cuda").bfloat16()
        step = K.PagesBatch(table, torch.tensor([0, m], dtype=torch.int32, device="cuda"), lens, m, m)
        out = torch.empty_like(q)
        store.attention_dev(step, q, heads, 0.1, out)
        x = torch.einsum("ihd,thd->iht", q.double(), k.double()) * 0.1
        t, p = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")
        x = x.masked_fill((t[None] > p[:, None])[:, None], -math.inf)
        w = torch.softmax(x, -1)
        o = torch.einsum("iht,thd->ihd", w, v.double())
        a = torch.einsum("iht,thd->ihd", w, v.double().abs())
        assert bool(((out.double() - o).abs() <= 2.0**-8 * o.abs() + 1.1 * 2.0**-8 * a).all())
    store.status()


def test_reported_batches(env):
    """Pages and lengths outside their arrays are clamped and reported once."""
    torch, K = env
    for spec in (DECODE[2], CHUNK[2]):
        c = Case(env, bits=16, **spec)
        q = c.queries()
        out = torch.empty_like(q)
        c.table[0, 0] = c.pages
        c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, out)
        with pytest.raises(K.KiviError) as e:
            c.store.status()
        assert e.value.variant == "InvalidArgument" and "page" in e.value.message
        c.store.status()
        c.table[0, 0] = 0
        c.kv_lens[0] = 1 << 30
        c.store.read_dev(c.step, *[torch.empty(c.total, c.heads, c.dim, dtype=c.dtype, device="cuda") for _ in range(2)])
        with pytest.raises(K.KiviError) as e:
            c.store.status()
        assert "lengths" in e.value.message


def test_nothing_to_do(env):
    torch, K = env
    c = Case(env, [0, 0], [30, 0], bits=8)
    q = torch.empty(0, c.heads * c.group, c.dim, dtype=c.dtype, device="cuda")
    c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, q)
    x = torch.empty(0, c.heads, c.dim, dtype=c.dtype, device="cuda")
    c.store.write_dev(c.step, x, x)
    c.store.read_dev(c.step, x, x)
    c.store.status()


def test_refusals(env):
    """Refused before anything is launched, output untouched."""
    torch, K = env
    c = Case(env, [1, 2], [30, 40], heads=2, group=2, dim=64)
    q = c.queries()
    out = torch.zeros_like(q)
    before = K.kernel_launches()

    def refused(variant, call):
        with pytest.raises(K.KiviError) as e:
            call()
        assert e.value.variant == variant, e.value

    attend = c.store.attention_dev
    refused("QueryHeads", lambda: attend(c.step, q[:, :3], 3, 0.1, out[:, :3]))
    refused("InvalidArgument", lambda: attend(c.step, q[:2], 4, 0.1, out))              # shape
    refused("InvalidArgument", lambda: attend(c.step, q, 4, 0.1, out.half()))           # types differ
    refused("InvalidArgument", lambda: attend(c.step, q.half(), 4, 0.1, out.half()))    # not the pages'
    refused("Unsupported", lambda: attend(c.step, q.float(), 4, 0.1, out.float()))
    refused("InvalidArgument", lambda: attend(c.step, q.mT.contiguous().mT, 4, 0.1, out))  # strided elements
    refused("InvalidArgument", lambda: attend(c.step, q, 4, 0.1, out[:, :1].expand(3, 4, 64)))  # rows overlap
    refused("InvalidArgument", lambda: attend(c.step, q, 4, 0.1, out, window=-1))
    refused("InvalidArgument", lambda: attend(c.step, q, 4, 0.1, out, d_lse=torch.zeros(3, 4)[:, ::2]))
    refused("InvalidArgument", lambda: attend(c.step, None, 4, 0.1, None, dtype="bf16"))
    refused("InvalidArgument", lambda: c.store.write_dev(c.step, q[:, :2], q[:, :2].half()))
    refused("InvalidArgument", lambda: c.store.write_dev(c.step, q, q))                 # four heads, not two
    refused("InvalidArgument", lambda: c.store.read_dev(c.step, out[:, :1].expand(3, 2, 64), out[:, :1].expand(3, 2, 64)))
    wide = torch.zeros(3, 2 * 257, 64, dtype=c.dtype, device="cuda")
    refused("Unsupported", lambda: attend(c.step, wide, 2 * 257, 0.1, wide))
    with pytest.raises(K.KiviError):
        K.KvPages(c.config, c.data[0][:1], c.data[1])                                   # too little memory
    assert K.kernel_launches() == before and bool((out == 0).all())


def test_handles_share_a_device(env):
    """Two stores attending in turn on two streams, and one freed between."""
    torch, K = env
    a, b = Case(env, seed=1, **CHUNK[3]), Case(env, bits=8, seed=2, **DECODE[6])
    qa, qb = a.queries(), b.queries()
    wa, wb = a.attend(qa, 0.1)[0], b.attend(qb, 0.1)[0]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(torch.empty_like(qa), torch.empty_like(qb)) for _ in range(8)]
    torch.cuda.synchronize()
    for oa, ob in outs:
        a.store.attention_dev(a.step, qa, a.heads * a.group, 0.1, oa, stream=s)
        b.store.attention_dev(b.step, qb, b.heads * b.group, 0.1, ob, stream=t)
    torch.cuda.synchronize()
    assert all(torch.equal(oa, wa) and torch.equal(ob, wb) for oa, ob in outs)
    a.store.close()
    assert torch.equal(b.attend(qb, 0.1)[0], wb)


def test_broadcast_inputs(env):
    """One row written to every token and head (strides 0)."""
    torch, K = env
    c = Case(env, [5], [5], heads=3, dim=32, bits=8)
    row = torch.randn(1, 1, 32, device="cuda").to(c.dtype)
    c.store.write_dev(c.step, row.expand(5, 3, 32), row.expand(5, 3, 32))
    k, v = torch.empty(5, 3, 32, dtype=c.dtype, device="cuda"), torch.empty(5, 3, 32, dtype=c.dtype, device="cuda")
    c.store.read_dev(c.step, k, v)
    assert bool((k == k[:1, :1]).all()) and torch.equal(k, v) and bool(((k - row).abs() <= 0.05).all())


def test_many_short_sequences(env):
    """More sequences than a CTA has threads, decode and chunks."""
    torch, K = env
    for new in ([1] * 700, [i % 4 for i in range(700)]):
        c = Case(env, new, [max(n, i % 37) for i, n in enumerate(new)], heads=1, group=2, dim=32)
        c.check(c.queries(), 0.2)


def test_example_runs(env):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kivi-cache-rs_b200", "examples",
                        "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for bits in (16, 8, 4):
        worst = mod.serve(bits=bits, sequences=3, prompt=150, steps=4, window=64, sinks=4, page_size=16)
        assert worst <= 0.05, (bits, worst)
