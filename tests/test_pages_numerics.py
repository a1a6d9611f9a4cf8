"""The paged store where its arithmetic and its shared state can go wrong: zeros,
infinities and values of unlike size beside one another, extreme windows, streams and
workspaces.  Cases, the 64-bit reference and its tolerances are test_pages.py's."""
import math

import pytest

from test_pages import Case, env  # noqa: F401  (env is a fixture)

pytestmark = pytest.mark.gpu


def rewrite(c, k=None, v=None):
    """The whole sequences again with other keys or values."""
    c.k = c.k if k is None else k.to(c.dtype)
    c.v = c.v if v is None else v.to(c.dtype)
    c.store.write_dev(c.whole, c.k, c.v)


# ------------------------------------------------------------------ zeros


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "bf16"), (8, "f16"), (4, "bf16")])
@pytest.mark.parametrize("q,k", [(0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (0.0, 1e-3), (1e-3, 0.0)])
@pytest.mark.parametrize("new", [1, 70])
def test_zero_queries_and_keys(env, bits, kind, q, k, new):
    """Scores of zero are equal weights for what a row sees."""
    c = Case(env, [new], [200], heads=1, bits=bits, kind=kind)
    rewrite(c, k=c.k * k)
    c.check(c.queries() * q, 0.1)
    c.check(c.queries() * q, 0.1, 33, 5)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("size", [0.25, 1e-4])
def test_scale_zero(env, bits, size):
    c = Case(env, [70], [200], heads=1, bits=bits)
    rewrite(c, k=c.k * size)
    c.check(c.queries() * size, 0.0)


# ------------------------------------------------------------------ values of unlike size


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "bf16"), (8, "f16"), (4, "bf16")])
@pytest.mark.parametrize("new", [1, 70, 300])
@pytest.mark.parametrize("sizes", [(1, 0), (100, 0), (1000, 0), (0, 1000), (1, 1000, 1e-3), (0, 0)])
def test_runs_of_unlike_values(env, bits, kind, new, sizes):
    """128 tokens of one size after 128 of another, zeros among them: outputs and
    log-sum-exps, causal and under a window."""
    torch, K = env
    c = Case(env, [new], [800], heads=1, bits=bits, kind=kind)
    t = torch.arange(800, device="cuda") // 128
    size = torch.tensor(sizes, device="cuda")[t % len(sizes)].float()
    rewrite(c, v=c.v * size[:, None, None])
    q = c.queries()
    c.check(q, 0.1)
    c.check(q, 0.1, 200, 140)


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "bf16"), (4, "bf16")])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("big", [1e6, 1e9, 1e12])
def test_large_values_of_small_weight(env, bits, kind, new, big):
    """Tokens whose values are far larger and whose weights are as much smaller: what
    the others give stays exact to its own size."""
    torch, K = env
    c = Case(env, [new], [640], heads=1, bits=bits, kind=kind)
    k, v = c.k.float() * 0.3, c.v.float()
    large = (torch.arange(640, device="cuda") // 128) % 2 == 0
    k[:, :, 0] = torch.where(large, -8.0, 0.0)[:, None]
    v[large] *= big
    rewrite(c, k=k, v=v)
    q = c.queries() * 0.3
    q[:, :, 0] = 1.0
    c.check(q, math.log(big * 1e3) / 8)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("sizes", [(1e30, 1e-8), (1e-30, 1e30), (1e30, 0, 1e-30, 1e30)])
@pytest.mark.parametrize("new", [1, 130])
def test_runs_of_extreme_values(env, bits, sizes, new):
    """Sums that no exponent of the small values holds."""
    torch, K = env
    c = Case(env, [new], [800], heads=1, bits=bits)
    t = torch.arange(800, device="cuda") // 128
    size = torch.tensor(sizes, device="cuda")[t % len(sizes)].float()
    rewrite(c, v=c.v.float() * size[:, None, None])
    c.check(c.queries(), 0.1)
    c.check(c.queries(), 0.1, 200, 140)


# ------------------------------------------------------------------ infinities and NaN


@pytest.mark.parametrize("bits,kind,bad", [(16, "bf16", math.inf), (16, "bf16", math.nan), (16, "f16", math.inf),
                                           (8, "bf16", math.inf), (4, "f16", math.inf)])
@pytest.mark.parametrize("at", range(8))
def test_a_score_that_is_not_finite(env, bits, kind, at, bad):
    """NaN in every channel of the rows that see it, nothing in the others', at each of
    eight neighbouring tokens (the codec leaves a NaN out of its row's range, so for codes
    an infinity, whose row's parameters are not finite)."""
    torch, K = env
    new, kv, row = 70, 200, 24 + at
    c = Case(env, [new], [kv], heads=1, bits=bits, kind=kind)
    q = c.queries()
    q[:, :, 3] = q[:, :, 3].abs() + 0.5
    want, wlse = c.attend(q, 0.1)
    k = c.k.clone()
    k[kv - new + row, 0, 3] = bad
    rewrite(c, k=k)
    got, lse = c.attend(q, 0.1)
    assert torch.equal(got[:row], want[:row]) and torch.equal(lse[:row], wlse[:row])
    assert bool(torch.isnan(got[row:]).all()) and bool(torch.isnan(lse[row:]).all())
    # out of the window again for the last rows
    got, _ = c.attend(q, 0.1, 16, 2)
    assert bool(torch.isnan(got[row:row + 16]).all())
    assert bool(torch.isfinite(got[row + 16:]).all()) and bool(torch.isfinite(got[:row]).all())


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_scores_that_overflow(env, bits):
    """Finite keys and queries whose product does not fit fp32."""
    torch, K = env
    for at in range(8):
        c = Case(env, [70], [200], heads=1, bits=bits)
        q = c.queries()
        q[:, :, 3] = 1e30
        k = c.k.clone()
        k[:, :, 3] = 0
        k[130 + 24 + at, 0, 3] = 1e30
        rewrite(c, k=k)
        got, _ = c.attend(q, 1.0)
        assert bool(torch.isnan(got[24 + at:]).all())
        assert not bool(torch.isnan(got[:24 + at]).any())


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (16, "f16"), (8, "bf16"), (4, "bf16")])
@pytest.mark.parametrize("new", [1, 70, 300])
@pytest.mark.parametrize("scale", [1e6, -1e6, 1e12, 1e25])
def test_scores_far_apart(env, bits, kind, new, scale):
    """Scores past what fp32 holds to the unit: all of a row's weight on its largest one,
    or shared by the tokens that tie."""
    torch, K = env
    c = Case(env, [new], [500], heads=1, bits=bits, kind=kind)
    k = torch.zeros_like(c.k)
    k[:, 0, 3] = (1 + torch.arange(500, device="cuda") * 37 % 61) / 61
    rewrite(c, k=k)
    q = torch.zeros_like(c.queries())
    q[:, :, 3] = 1.0 + torch.arange(4, device="cuda") / 4
    for window, sinks in ((0, 0), (150, 3)):
        out, _ = c.attend(q, scale, window, sinks)
        held = [x[0] for x in (c.held(0), c.held(1))]
        for i in range(new):
            p = 500 - new + i
            t = torch.arange(500, device="cuda")
            see = (t <= p) & ((t > p - window) | (t < sinks) if window else t >= 0)
            x = held[0][:, 0, 3] * (1 if scale > 0 else -1)
            x[~see] = -math.inf
            ties = x >= x.max() - 1e-3
            v = held[1][ties, 0]
            u = 2.0**-8 if kind == "bf16" else 2.0**-11
            tol = (2 * u + 2.0**-10) * v.abs().mean(0) + 2.0**-16
            assert bool(((out[i].double() - v.mean(0)).abs() <= tol).all())


@pytest.mark.parametrize("at", range(8))
@pytest.mark.parametrize("big", [1e38, -3e38])
def test_a_token_out_of_sight_weighs_nothing(env, at, big):
    """The largest bf16 values in a newest token, and behind the window: rows that do not
    see them keep every bit."""
    torch, K = env
    new, kv, row = 70, 200, 24 + at
    c = Case(env, [new], [kv], heads=1)
    q = c.queries()
    v = c.v.clone()
    v[kv - new + row] = big
    want, _ = c.attend(q, 0.1)
    wide, _ = c.attend(q, 0.1, 16, 2)
    rewrite(c, v=v)
    got, _ = c.attend(q, 0.1)
    assert torch.equal(got[:row], want[:row])
    got, _ = c.attend(q, 0.1, 16, 2)
    assert torch.equal(got[:row], wide[:row]) and torch.equal(got[row + 16:], wide[row + 16:])


# ------------------------------------------------------------------ windows


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", [(2**31 - 1, 0), (2**31 - 1, 3), (2**31 - 4, 0), (1 << 40, 2**31 - 1), (2**31 - 300, 5)])
@pytest.mark.parametrize("new,kv", [([8], [5]), ([300, 1], [290, 40]), ([70], [200]), ([1], [200])])
def test_windows_as_large_as_none(env, bits, window, sinks, new, kv):
    """Also where more tokens are new than the cache counts, so that rows stand before it."""
    torch, K = env
    c = Case(env, new, kv, heads=1, bits=bits)
    q = c.queries()
    want, wlse = c.attend(q, 0.1)
    got, lse = c.check(q, 0.1, window, sinks)
    assert torch.equal(got, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("side", ["keys", "values", "both"])
@pytest.mark.parametrize("big", [1e6, 1e12, 1e38])
@pytest.mark.parametrize("at", [0, 1, 24, 69])
def test_a_token_out_of_sight_takes_no_precision(env, bits, side, big, at):
    """Codes: huge keys or values in one newest token leave the rows that do not see it
    as exact as before; those that do see it are right too."""
    torch, K = env
    new, kv = 70, 200
    c = Case(env, [new], [kv], heads=1, bits=bits)
    k, v = c.k.float(), c.v.float()
    x = kv - new + at
    if side != "values":
        k[x] = k[x].sign() * big
    if side != "keys":
        v[x] = v[x].sign() * big
    rewrite(c, k=k, v=v)
    q = c.queries()
    for window, sinks in ((0, 0), (16, 2)):
        out, lse = c.attend(q, 0.1, window, sinks)
        o, l, tol, ltol = c.reference(q, 0.1, window, sinks)
        hidden = torch.ones(new, dtype=torch.bool, device="cuda")
        hidden[at:at + window if window else new] = False
        assert bool(((out.double() - o).abs() <= tol)[hidden].all())
        assert bool(((lse.double() - l).abs() <= ltol)[hidden].all())
        if side == "values":
            assert bool(((out.double() - o).abs() <= tol)[~hidden].all())
        else:  # one weight is all of them, or nothing
            assert bool(torch.isfinite(out[~hidden]).all())


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("at", [0, 5, 24, 63])
def test_a_value_that_is_not_finite(env, bits, at):
    """An infinite value among a newest token's: its channel in the rows that see it (codes:
    every channel, since the row's parameters are not finite), every other output as exact."""
    torch, K = env
    new, kv = 70, 200
    c = Case(env, [new], [kv], heads=1, bits=bits)
    q = c.queries()
    v = c.v.clone()
    v[kv - new + at, 0, 5] = math.inf
    rewrite(c, v=v)
    out, lse = c.attend(q, 0.1)
    o, l, tol, ltol = c.reference(q, 0.1)
    assert bool(((lse.double() - l).abs() <= ltol).all())
    good = torch.ones(out.shape, dtype=torch.bool, device="cuda")
    good[at:, :, 5 if bits == 16 else slice(None)] = False
    assert bool(((out.double() - o).abs() <= tol)[good].all())
    assert not bool(torch.isfinite(out[~good]).any())


# ------------------------------------------------------------------ shared state


def test_threads_on_their_default_streams(env):
    """cudaStreamPerThread is one handle for a stream of each host thread: two threads'
    calls share the device's scratch safely."""
    import threading

    torch, K = env
    cases = [Case(env, [1], [20011], heads=1, group=5, seed=1), Case(env, [300], [4000], heads=1, group=4, page=64, seed=2)]
    queries = [c.queries() for c in cases]
    want = [c.attend(q, 0.1)[0] for c, q in zip(cases, queries)]
    outs = [[torch.empty_like(q) for _ in range(40)] for q in queries]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            c = cases[i]
            for o in outs[i]:
                c.store.attention_dev(c.step, queries[i], c.heads * c.group, 0.1, o, stream=2)
        except Exception as e:  # noqa: BLE001  (reported by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for w, o in zip(want, outs):
        assert all(torch.equal(x, w) for x in o)


def test_streams_made_anew(env):
    """A stream that is gone and one with its handle are two streams."""
    import ctypes as C

    torch, K = env
    rt = C.CDLL("libcudart.so.12")
    c = Case(env, [1], [20011], heads=1, group=5)
    q = c.queries()
    want, _ = c.attend(q, 0.1)
    outs = [torch.empty_like(q) for _ in range(60)]
    torch.cuda.synchronize()
    for o in outs:
        s = C.c_void_p()
        assert rt.cudaStreamCreateWithFlags(C.byref(s), 1) == 0  # non-blocking
        c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, o, stream=s.value)
        assert rt.cudaStreamDestroy(s) == 0  # its work goes on
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_a_new_store_on_a_busy_device(env):
    """A handle made while the default stream is busy is ready when it is returned: what
    another stream's call reports is not cleared later."""
    torch, K = env
    c = Case(env, [1], [40], heads=1)
    q, s = c.queries(), torch.cuda.Stream()
    out = torch.empty_like(q)
    c.table[0, 0] = -1
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    store = K.KvPages(c.config, *c.data)
    store.attention_dev(c.step, q, c.group, 0.1, out, stream=s)
    s.synchronize()
    with pytest.raises(K.KiviError) as e:
        store.status()
    assert "page" in e.value.message
    store.status()


def test_graphs_with_workspaces_beside_one_another(env):
    """Two captured steps, each with a workspace of its own, replayed on two streams beside
    live calls on a third."""
    torch, K = env
    specs = [dict(new=[1], kv=[20011], group=5, heads=1), dict(new=[300], kv=[4000], group=4, heads=1, page=64)]
    cases = [Case(env, seed=i, **s) for i, s in enumerate(specs + specs[:1])]
    queries = [c.queries() for c in cases]
    want = [c.attend(q, 0.1)[0] for c, q in zip(cases, queries)]
    outs, graphs, streams = [torch.empty_like(q) for q in queries], [], [torch.cuda.Stream() for _ in range(3)]
    for c, q, o, s in zip(cases[:2], queries, outs, streams):
        c.store.set_workspace(torch.empty(K.pages_workspace_size() // 4, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.store.attention_dev(c.step, q, c.heads * c.group, 0.1, o, stream=s)
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            c = cases[2]
            c.store.attention_dev(c.step, queries[2], c.heads * c.group, 0.1, outs[2], stream=streams[2])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    for c in cases:
        c.store.status()


def test_a_report_readies_the_workspace(env):
    """Counters that a call left raised are cleared with its report."""
    torch, K = env
    c = Case(env, [1], [20011], heads=1, group=5)
    q = c.queries()
    want, _ = c.attend(q, 0.1)
    w = torch.empty(K.pages_workspace_size() // 4, dtype=torch.int32, device="cuda").fill_(7)
    c.store.set_workspace(w)
    assert bool((w[-2048:] == 0).all())
    w[-2048:] = 1
    c.kv_lens[0] = 1 << 30
    c.store.read_dev(c.step, *[torch.empty(1, 1, 128, dtype=c.dtype, device="cuda") for _ in range(2)])
    with pytest.raises(K.KiviError) as e:
        c.store.status()
    assert "lengths" in e.value.message and bool((w[-2048:] == 0).all())
    c.kv_lens[0] = 20011
    assert torch.equal(c.attend(q, 0.1)[0], want)
    c.store.set_workspace(None)
    assert torch.equal(c.attend(q, 0.1)[0], want)
    for bad in (w[:100], w.cpu(), torch.empty(2, w.numel(), dtype=torch.int32, device="cuda").T):
        with pytest.raises(K.KiviError):
            c.store.set_workspace(bad)
    with pytest.raises(K.KiviError):
        c.store.set_workspace(w.data_ptr() + 4, 4 * w.numel())
    assert torch.equal(c.attend(q, 0.1)[0], want)


def test_rows_without_sequences_are_refused(env):
    """Rows that no call could fill are an error, not outputs left as they were."""
    torch, K = env
    c = Case(env, [3, 2], [30, 40], heads=2)
    q = c.queries()
    out = torch.zeros_like(q)
    k, v = torch.zeros(5, 2, 128, dtype=c.dtype, device="cuda"), torch.zeros(5, 2, 128, dtype=c.dtype, device="cuda")
    before = K.kernel_launches()
    for batch in (c.batch(c.cu, 5, 0), K.PagesBatch(c.table, c.cu, c.kv_lens, 5, 3, batch=0)):
        for call in (lambda: c.store.attention_dev(batch, q, 8, 0.1, out), lambda: c.store.write_dev(batch, k, v),
                     lambda: c.store.read_dev(batch, k, v)):
            with pytest.raises(K.KiviError) as e:
                call()
            assert e.value.variant == "InvalidArgument" and "rows" in e.value.message
    assert K.kernel_launches() == before
    c.store.status()


@pytest.mark.parametrize("new", [[3, 2], [1, 1]])
def test_rows_of_nobody_are_left_alone(env, new):
    """A step padded to more rows than its sequences have."""
    torch, K = env
    c = Case(env, new, [30, 40], heads=2)
    n = sum(new)
    want, _ = c.attend(c.queries(), 0.1)
    step = c.batch(c.cu, n + 3, max(new))
    q = torch.zeros(n + 3, 8, 128, dtype=c.dtype, device="cuda")
    c.g.manual_seed(5)
    q[:n] = c.queries()
    out = torch.full_like(q, 7.0)
    c.store.attention_dev(step, q, 8, 0.1, out)
    assert torch.equal(out[:n], c.attend(q[:n].contiguous(), 0.1)[0]) and bool((out[n:] == 7).all())
    k, v = torch.full((n + 3, 2, 128), 7.0, dtype=c.dtype, device="cuda"), torch.empty(n + 3, 2, 128, dtype=c.dtype, device="cuda")
    c.store.read_dev(step, k, v)
    assert bool((k[n:] == 7).all()) and not bool((k[:n] == 7).all())
    c.store.status()


def test_interleaved_outputs(env):
    """Any strides whose rows do not meet are taken; where a token one way and a head back
    meet, the call is refused."""
    torch, K = env
    c = Case(env, [5], [40], heads=2, dim=64)
    q = c.queries()  # [5, 8, 64]
    want, _ = c.attend(q, 0.1)
    room = torch.zeros(1 << 16, dtype=c.dtype, device="cuda")

    def meet(rows, heads, token, head):
        at = sorted(t * token + h * head for t in range(rows) for h in range(heads))
        return any(b - a < 64 for a, b in zip(at, at[1:]))

    strides = [(64, 64), (64, 128), (128, 64), (512, 64), (64, 320), (500, 64), (511, 72), (192, 320), (64 * 9, 64 * 2), (64 * 2, 64 * 9),
               (96, 640), (128, 192), (320, 320), (640, 79), (640, 80), (1000, 64), (130, 650), (65, 325), (64 * 3, 64 * 16)]
    taken = 0
    for token, head in strides:
        out = room.as_strided((5, 8, 64), (token, head, 1))
        if meet(5, 8, token, head):
            with pytest.raises(K.KiviError) as e:
                c.store.attention_dev(c.step, q, 8, 0.1, out)
            assert e.value.variant == "InvalidArgument" and "overlap" in e.value.message
        else:
            c.store.attention_dev(c.step, q, 8, 0.1, out)
            assert torch.equal(out, want)
            taken += 1
    assert 6 <= taken <= len(strides) - 6


@pytest.mark.parametrize("bits,kind", [(16, "f16"), (16, "bf16"), (8, "f16"), (4, "bf16")])
@pytest.mark.parametrize("new", [1, 2])
def test_many_small_weights(env, bits, kind, new):
    """One token holds almost all of the weight and no value, as first tokens do; the sum of
    3000 others, 2^-23 of it each, is the output.  As many sequences as fill the device, so
    that one row's tiles meet in one sum.  An f16 weight is exact to 2^-32 of its row's
    largest, whatever bits that leaves it."""
    torch, K = env
    n, seqs = 3000, 150
    c = Case(env, [new] * seqs, [n] * seqs, heads=1, group=4, bits=bits, kind=kind, page=64)
    k, v = torch.zeros_like(c.k), torch.ones_like(c.v)
    v[:, :, ::2] = 0.5
    k[::n, 0, 0], v[::n] = 16.0, 0.0
    rewrite(c, k=k, v=v)
    q = torch.zeros_like(c.queries())
    q[:, :, 0] = 1.0
    for log2 in (20.3, 22.6, 23.4):
        scale = log2 * math.log(2) / 16
        out, lse = c.attend(q, scale)
        o, l, tol, ltol = c.reference(q, scale)
        assert bool(((out.double() - o).abs() <= tol + n * 2.0**-32).all())
        assert bool(((lse.double() - l).abs() <= ltol).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new,window,sinks", [([130], 0, 0), ([37, 64, 130], 5, 4), ([300], 64, 0), ([3], 0, 0)])
@pytest.mark.parametrize("spread", [2.0, 3.0, 6.0])
def test_tokens_of_unlike_size(env, bits, new, window, sinks, spread):
    """Codes: values of 10^+-spread from token to token, and keys as unlike, seen and not."""
    torch, K = env
    c = Case(env, new, [n + 400 for n in new], heads=1, bits=bits)
    size = torch.rand(c.v.shape[0], 2, 1, 1, generator=c.g, device="cuda") * 2 - 1
    rewrite(c, k=c.k.float() * 10 ** (spread * (size[:, 0] - 1)), v=c.v.float() * 10 ** (spread * size[:, 1]))
    c.check(c.queries(), 0.3, window, sinks)
