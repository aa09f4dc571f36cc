"""The paged-cache operators as a program uses them: a run of all three over the steps of a stream, captured and replayed graphs, other
streams than the default one, two threads, and torch tensors (in a process of its own, on the runtime inside the PyTorch wheel)."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _hip():
    from hip_mem import hip
    h = hip()
    if not getattr(h, "paged_ready", False):
        vp = C.c_void_p
        h.hipStreamCreateWithFlags.argtypes = [C.POINTER(vp), C.c_uint]
        h.hipStreamSynchronize.argtypes = [vp]
        h.hipStreamDestroy.argtypes = [vp]
        h.hipStreamBeginCapture.argtypes = [vp, C.c_int]
        h.hipStreamEndCapture.argtypes = [vp, C.POINTER(vp)]
        h.hipGraphInstantiate.argtypes = [C.POINTER(vp), vp, C.POINTER(vp), vp, C.c_size_t]
        h.hipGraphLaunch.argtypes = [vp, vp]
        h.hipGraphExecDestroy.argtypes = [vp]
        h.hipGraphDestroy.argtypes = [vp]
        h.paged_ready = True
    return h


class Stream:
    def __init__(self):
        self.p = C.c_void_p()
        assert _hip().hipStreamCreateWithFlags(C.byref(self.p), 1) == 0      # not ordered with the default stream

    def sync(self):
        assert _hip().hipStreamSynchronize(self.p) == 0

    def close(self):
        _hip().hipStreamDestroy(self.p)


class Loop:
    """A small server's buffers: n requests, grouped heads, pages dealt out by the plan from one free list."""

    def __init__(self, n=3, heads=4, kvh=2, dim=64, page=16, pages=60, width=14, rows=64, window=0, sinks=0, kind="bfloat16", seed=0):
        import ptts_paged
        self.n, self.heads, self.kvh, self.dim, self.page, self.pages, self.width, self.rows = n, heads, kvh, dim, page, pages, width, rows
        self.window, self.sinks, self.kind = window, sinks, kind
        rng = np.random.default_rng(seed)
        self.order = rng.permutation(pages)
        self.taken = 0
        self.length = np.zeros(n, np.int64)
        self.freq = ptts_paged.frequencies(dim)[0]
        self.d = {k: ref.Dev(np.zeros(s), "int32") for k, s in dict(cached=n, arriving=n, slots=rows, positions=rows, cu=n + 1, kv_len=n, counts=4, status=1).items()}
        self.d["table"] = ref.Dev(np.full((n, width), -1), "int32")
        self.d["free"] = ref.Dev(np.full(pages, -1), "int32")
        self.d["freq"] = ref.Dev(self.freq, "float64")
        for k, s in dict(q=(rows, heads, dim), k=(rows, kvh, dim), v=(rows, kvh, dim), q_out=(rows, heads, dim), out=(rows, heads, dim),
                         kp=(pages, page, kvh, dim), vp=(pages, page, kvh, dim)).items():
            self.d[k] = ref.floats(np.zeros(s), kind)
        self.d["lse"] = ref.Dev(np.zeros((rows, heads)), "float32")
        self.d["ws"] = ref.Dev(np.zeros(1 << 22), "uint8")
        self.keys = [np.zeros((0, kvh, dim)) for _ in range(n)]
        self.values = [np.zeros((0, kvh, dim)) for _ in range(n)]

    def feed(self, arriving, rng):
        """New rows of a step on their way to the device."""
        self.arriving = np.asarray(arriving)
        fresh = int((-(-(self.length + arriving) // self.page) + (-self.length // self.page)).sum())
        free = np.full(self.pages, -1)
        free[:fresh] = self.order[self.taken:self.taken + fresh]
        self.taken += fresh
        self.x = {k: ref.rounded(rng.standard_normal((self.rows, h, self.dim)), self.kind) for k, h in (("q", self.heads), ("k", self.kvh), ("v", self.kvh))}
        for k, v in dict(cached=self.length, arriving=arriving, free=free).items():
            self.d[k].put(v)
        for k, v in self.x.items():
            self.d[k].put(ref.to_bits(v, self.kind))

    def launch(self, stream=None):
        import ptts_paged
        from ptts_paged import DeviceArray
        a = {k: v.a for k, v in self.d.items()}
        ws = DeviceArray(self.d["ws"].ptr, (1 << 20,), "int32")
        ptts_paged.plan(a["cached"], a["arriving"], a["free"], a["table"], self.page, slot_map=a["slots"], positions=a["positions"], cu_rows=a["cu"],
                        kv_len=a["kv_len"], counts=a["counts"], status=a["status"], stream=stream)
        # rows behind the new ones of this step name slot -1
        ptts_paged.rotary_append(a["q"], a["k"], a["v"], a["positions"], a["freq"], q_out=a["q_out"], slot_map=a["slots"], k_pages=a["kp"], v_pages=a["vp"],
                                 status=a["status"], stream=stream)
        ptts_paged.attention(a["q_out"], a["kp"], a["vp"], a["table"], a["cu"], a["kv_len"], out=a["out"], lse=a["lse"], window=self.window, sinks=self.sinks,
                             workspace=ws, status=a["status"], stream=stream)

    def check(self):
        """Against float64 from the rows as they were fed, one rounding where the device keeps a rotated row."""
        live = int(self.arriving.sum())
        pos = np.concatenate([self.length[i] + np.arange(self.arriving[i]) for i in range(self.n)]).astype(np.int64)
        q = ref.from_bits(self.d["q_out"].host(), self.kind)
        want_q = ref.rotate(self.x["q"][:live].astype(np.float64), pos, self.freq, False)
        assert (np.abs(q[:live] - want_q) <= ref.EPS[self.kind] * np.abs(want_q) + 1e-5).all()
        kp, vp = (ref.from_bits(self.d[k].host(), self.kind) for k in ("kp", "vp"))
        table = self.d["table"].host()
        cu = np.concatenate([[0], np.cumsum(self.arriving)])
        rk = ref.rotate(self.x["k"][:live].astype(np.float64), pos, self.freq, False)
        total = self.length + self.arriving
        for i in range(self.n):
            self.keys[i] = np.concatenate([self.keys[i], rk[cu[i]:cu[i + 1]]])
            self.values[i] = np.concatenate([self.values[i], self.x["v"][cu[i]:cu[i + 1]].astype(np.float64)])
            j = np.arange(total[i])
            got_k, got_v = kp[table[i, j // self.page], j % self.page], vp[table[i, j // self.page], j % self.page]
            assert (np.abs(got_k - self.keys[i]) <= ref.EPS[self.kind] * np.abs(self.keys[i]) + 1e-5).all()
            np.testing.assert_array_equal(got_v, self.values[i])
        # attention of what the pages and the rotated rows hold
        pick = [(lambda i, x=x: x[table[i, np.arange(total[i]) // self.page], np.arange(total[i]) % self.page]) for x in (kp, vp)]
        out, lse, size, logit = ref.attention(q[:live], pick[0], pick[1], cu, total, self.dim ** -0.5, self.window, self.sinks)
        b_out, b_lse = ref.attention_bounds(out, size, logit, lse, self.kind, self.dim, int(total.max()))
        assert (np.abs(ref.from_bits(self.d["out"].host(), self.kind)[:live] - out) <= b_out).all()
        assert (np.abs(self.d["lse"].host()[:live] - lse) <= b_lse).all()
        assert self.d["status"].host()[0] == 0 and self.d["counts"].host().tolist()[0] == live
        self.length = total


STEPS = [(20, 7, 31), (1, 1, 1), (0, 33, 1), (1, 1, 1), (16, 0, 16), (1, 1, 1), (1, 1, 1)]


def _clear_slots(loop):
    loop.d["slots"].put(np.full(loop.rows, -1))
    loop.d["positions"].put(np.zeros(loop.rows))


@pytest.mark.parametrize("window,sinks,kind", [(0, 0, "bfloat16"), (30, 4, "float16"), (0, 0, "float32")])
def test_run_of_steps(window, sinks, kind):
    loop, rng = Loop(window=window, sinks=sinks, kind=kind), np.random.default_rng(1)
    for a in STEPS:
        loop.feed(a, rng)
        _clear_slots(loop)
        loop.launch()
        loop.check()


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_captured_and_replayed(kind):
    """One graph of all three calls, replayed over steps of other lengths, with eager work and waits between."""
    h, s = _hip(), Stream()
    loop, eager, rng = Loop(kind=kind), Loop(kind=kind), np.random.default_rng(2)
    graph, run = C.c_void_p(), C.c_void_p()
    assert h.hipStreamBeginCapture(s.p, 1) == 0           # thread-local
    loop.launch(stream=s.p.value)
    assert h.hipStreamEndCapture(s.p, C.byref(graph)) == 0
    assert h.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
    for a in STEPS:
        state = rng.bit_generator.state
        loop.feed(a, rng)
        rng.bit_generator.state = state
        eager.feed(a, rng)
        _clear_slots(loop)
        _clear_slots(eager)
        eager.launch()
        assert h.hipGraphLaunch(run, s.p) == 0
        s.sync()
        for k in ("table", "slots", "positions", "cu", "kv_len", "counts", "q_out", "kp", "vp", "out", "lse"):
            np.testing.assert_array_equal(loop.d[k].host(), eager.d[k].host(), err_msg=k)
        loop.check()
        eager.check()
    h.hipGraphExecDestroy(run)
    h.hipGraphDestroy(graph)
    s.close()


def test_two_threads_on_two_streams():
    """Calls from two threads at once, each with its stream and workspace."""
    loops = [Loop(seed=i) for i in range(2)]
    errors = []

    def work(i):
        try:
            s, rng = Stream(), np.random.default_rng(10 + i)
            for a in STEPS:
                loops[i].feed(a, rng)
                _clear_slots(loops[i])
                loops[i].launch(stream=s.p.value)
                s.sync()
                loops[i].check()
            s.close()
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_offsets_beyond_32_bits():
    """Rows of a pool that lie more than 2^32 elements from its start."""
    import ptts_paged
    from ptts_paged import DeviceArray
    page, kvh, dim, heads = 16, 1, 64, 2
    far = (1 << 32) // 64 + 4096                                   # page stride in elements: page 70 lies beyond 2^32
    pages = 70
    total = (pages - 1) * far + page * dim
    p = [C.c_void_p() for _ in range(2)]
    for x in p:
        assert _hip().hipMalloc(C.byref(x), total * 2) == 0
    try:
        shape, strides = (pages, page, kvh, dim), (far, dim, dim, 1)
        kp, vp = (DeviceArray(x.value, shape, "bfloat16", strides) for x in p)
        rng = np.random.default_rng(0)
        n = 40
        k, v, q = (ref.rounded(rng.standard_normal((n, h, dim)), "bfloat16") for h in (kvh, kvh, heads))
        table = np.array([[69, 3, 68]])
        j = np.arange(n)
        d = [ref.floats(x, "bfloat16") for x in (k, v, q)]
        ints = {a: ref.Dev(b, "int32") for a, b in dict(slots=table[0, j // page] * page + j % page, pos=np.zeros(n), table=table, cu=[0, n], kl=[n], st=[0]).items()}
        freq, ws = ref.Dev(np.ones(1), "float64"), ref.Dev(np.zeros(1 << 20), "uint8")
        ptts_paged.rotary_append(None, d[0].a, d[1].a, ints["pos"].a, freq.a, slot_map=ints["slots"].a, k_pages=kp, v_pages=vp, status=ints["st"].a)
        for m in (n, 1):                                            # the chunk form, then a single row
            out, cu = ref.floats(np.zeros((n, heads, dim)), "bfloat16"), ref.Dev([0, m], "int32")
            ptts_paged.attention(d[2].a, kp, vp, ints["table"].a, cu.a, ints["kl"].a, out=out.a, max_rows=m, workspace=DeviceArray(ws.ptr, (1 << 18,), "int32"),
                                 status=ints["st"].a)
            want = ref.attention(q[:m], lambda i: k, lambda i: v, [0, m], [n], dim ** -0.5)
            bound, _ = ref.attention_bounds(want[0], want[2], want[3], want[1], "bfloat16", dim, n)
            assert (np.abs(ref.from_bits(out.host(), "bfloat16")[:m] - want[0]) <= bound).all()
        assert ints["st"].host()[0] == 0
    finally:
        for x in p:
            _hip().hipFree(x)


TORCH = r'''
import sys
sys.path[:0] = [%(pyhost)r]
import torch
import ptts_lib, ptts_paged as P
torch.manual_seed(0)
dev = "cuda"
n, heads, kvh, dim, page, rows = 5, 8, 2, 128, 16, 300
cached = torch.tensor([0, 37, 200, 64, 5000], dtype=torch.int32, device=dev)
arriving = torch.tensor([90, 1, 130, 0, 1], dtype=torch.int32, device=dev)
live = int(arriving.sum())
have, end = (cached + page - 1) // page, (cached + arriving + page - 1) // page
order = torch.randperm(int(end.sum()) + 9, device=dev).int()
table = torch.full((n, int(end.max()) + 1), -1, dtype=torch.int32, device=dev)
at = 0
for i in range(n):
    table[i, :int(have[i])] = order[at:at + int(have[i])]
    at += int(have[i])
free = order[at:]
z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=dev)
slots, pos, cu, kl, counts, status = torch.full((rows,), -1, dtype=torch.int32, device=dev), z(rows), z(n + 1), z(n), z(4), z(1)
bf = torch.bfloat16
qkv = torch.randn(rows, heads + 2 * kvh, dim, device=dev, dtype=bf)
pool = torch.randn(len(order), 2, page, kvh, dim, device=dev, dtype=bf)
kp, vp = pool[:, 0], pool[:, 1]
freq = torch.from_numpy(P.frequencies(dim)[0]).to(dev)
q_out, out, lse = z(rows, heads, dim, dt=bf), z(rows, heads, dim, dt=bf), z(rows, heads, dt=torch.float32)

def step():
    P.plan(cached, arriving, free, table, page, slot_map=slots, positions=pos, cu_rows=cu, kv_len=kl, counts=counts, status=status)
    P.rotary_append(qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:], pos, freq, q_out=q_out, slot_map=slots, k_pages=kp, v_pages=vp, status=status)
    P.attention(q_out, kp, vp, table, cu, kl, out=out, lse=lse, status=status)

def check(what):
    torch.cuda.synchronize()
    assert int(status) == 0 and counts.tolist()[0] == live, (what, status, counts)
    angle = pos[:live].double()[:, None] * freq
    x = qkv[:live].double()
    a, b, c, s = x[..., :dim // 2], x[..., dim // 2:], angle.cos()[:, None], angle.sin()[:, None]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    assert (q_out[:live].double() - turned[:, :heads]).abs().max() < 2.0 ** -8 * turned.abs().max(), what
    flat_k, flat_v = kp.reshape(-1, kvh, dim), vp.reshape(-1, kvh, dim)
    assert torch.equal(flat_v[slots[:live].long()], qkv[:live, heads + kvh:]), what
    assert (flat_k[slots[:live].long()].double() - turned[:, heads:heads + kvh]).abs().max() < 2.0 ** -8 * turned.abs().max(), what
    for i in range(n):
        L, lo, hi = int(kl[i]), int(cu[i]), int(cu[i + 1])
        j = torch.arange(L, device=dev)
        idx = table[i, j // page].long() * page + j %% page
        K, V = flat_k[idx].double(), flat_v[idx].double()
        for h in range(heads):
            w = q_out[lo:hi, h].double() @ K[:, h // 4].T * dim ** -0.5
            p = torch.arange(L - (hi - lo), L, device=dev)[:, None]
            w = w.masked_fill(j[None] > p, float("-inf"))
            want = torch.softmax(w, -1) @ V[:, h // 4]
            # half a step for the weights, half a step for the result
            bound = 2.0 ** -8 * (torch.softmax(w, -1) @ V[:, h // 4].abs() + want.abs()) + 1e-4
            assert ((out[lo:hi, h].double() - want).abs() <= bound).all(), (what, i, h)
            assert (lse[lo:hi, h].double() - torch.logsumexp(w, -1)).abs().max() < 1e-4 if hi > lo else True, (what, i, h)
    assert not out[live:].any()

step()
assert ptts_lib.runtime == "torch"
check("default stream")
s = torch.cuda.Stream()
out.zero_(); q_out.zero_()
s.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(s):
    step()
torch.cuda.current_stream().wait_stream(s)
check("another stream")
g = torch.cuda.CUDAGraph()
s.wait_stream(torch.cuda.current_stream())
with torch.cuda.graph(g, stream=s):
    step()
for _ in range(3):
    qkv.copy_(torch.randn_like(qkv))
    slots.fill_(-1)
    out.zero_(); q_out.zero_()
    g.replay()
    check("graph")
want = out.clone()
out.zero_()
P.attention(q_out, kp, vp, table, cu, kl, out=out, lse=lse, stream=torch.cuda.current_stream())
torch.cuda.synchronize()
assert torch.equal(out, want)
for bad in (lambda: P.attention(q_out.cpu(), kp, vp, table, cu, kl, out=out), lambda: P.attention(q_out, kp, vp, table.long(), cu, kl, out=out),
            lambda: P.attention(q_out, kp, vp, table, cu, kl, out=out, workspace=z(1)), lambda: P.attention(q_out, kp, vp, table, cu, kl, out=out.float()),
            lambda: P.attention(q_out, kp, vp, table, cu, kl, out=out, stream="x")):
    try:
        bad()
    except ptts_lib.PttsError as e:
        print("refused:", e)
    else:
        raise AssertionError("not refused")
try:
    P.attention(q_out, kp)
except TypeError as e:
    print("refused:", e)
import ptts_pack as pp
import os, tempfile, numpy as np
path = os.path.join(tempfile.gettempdir(), f"ptts_torch_{os.getpid()}.ptts")
pp.make_pack(path, pp.Spec.tiny(), seed=7, eos_bias=-20.0, layer_scale=0.2)
eng = ptts_lib.Engine(path, precision="fp32", temperature=0.0, lsd_steps=2, max_frames=4)          # the engine on the same runtime
r = eng.generate_ids([np.arange(5)], [np.zeros((3, eng.d_model), np.float32)])[0]
assert r["frames"] == 4 and np.isfinite(r["audio"]).all()
eng.close()
os.unlink(path)
print("TORCH OK")
'''


def test_torch_tensors(tmp_path):
    script = tmp_path / "torch_run.py"
    script.write_text(TORCH % dict(pyhost=os.path.join(ROOT, "pocket-tts.cpp_amd", "pyhost")))
    r = subprocess.run([sys.executable, "-u", str(script)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "TORCH OK" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
    assert r.stdout.count("refused:") == 6


def test_device_out_of_range_is_refused():
    import ptts_lib
    import ptts_paged
    from ptts_paged import DeviceArray
    a = {k: DeviceArray(1 << 20, (1,) if k != "t" else (1, 4), "int32", None, 99) for k in ("c", "n", "f", "t", "s", "p", "k")}
    with pytest.raises(ptts_lib.PttsError, match="device 99"):
        ptts_paged.plan(a["c"], a["n"], a["f"], a["t"], 16, slot_map=a["s"], positions=a["p"], cu_rows=DeviceArray(1 << 20, (2,), "int32", None, 99),
                        kv_len=a["k"], counts=DeviceArray(1 << 20, (4,), "int32", None, 99))
    loop = Loop()                                           # and the next call runs
    loop.feed((1, 2, 3), np.random.default_rng(0))
    _clear_slots(loop)
    loop.launch()
    loop.check()


def _one_request(kind, q, k, v, new, splits_wanted=True):
    """Attention of the last `new` rows of one sequence, pages in order; returns out, lse."""
    import ptts_paged
    from ptts_paged import DeviceArray
    n, kvh, dim = k.shape
    page = 16
    pages = -(-n // page)
    pad = [(0, pages * page - n), (0, 0), (0, 0)]
    d = [ref.floats(q, kind)] + [ref.floats(np.pad(x, pad).reshape(pages, page, kvh, dim), kind) for x in (k, v)]
    out, lse = ref.floats(np.zeros(q.shape), kind), ref.Dev(np.zeros(q.shape[:2]), "float32")
    ints = [ref.Dev(x, "int32") for x in (np.arange(pages)[None], [0, new], [n], [0])]
    a = [x.a for x in d] + [x.a for x in ints[:3]]
    need = ptts_paged.attention_workspace(*a, out=out.a, max_rows=new)
    ws = ref.Dev(np.full(max(need, 16), 255), "uint8")
    ptts_paged.attention(*a, out=out.a, lse=lse.a, max_rows=new, workspace=DeviceArray(ws.ptr, (max(need, 16) // 4,), "int32"), status=ints[3].a)
    assert ints[3].host()[0] == 0 and (need > 0) == splits_wanted
    return ref.from_bits(out.host(), kind), lse.host()


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n,new,splits", [(300, 1, False), (9000, 1, True), (300, 40, False), (9000, 40, True)])
def test_queries_that_are_nan(kind, n, new, splits):
    """A query of NaN gives NaN, in the row that holds it alone; so does a NaN that all keys of one wave hold."""
    rng = np.random.default_rng(n + new)
    q, k, v = (ref.rounded(rng.standard_normal((m, h, 64)), kind) for m, h in ((new, 2), (n, 1), (n, 1)))
    splits = splits or (kind == "float32" and n > 4000)
    q[0, 0, 5] = np.nan
    out, lse = _one_request(kind, q, k, v, new, splits)
    assert np.isnan(out[0, 0]).all() and np.isnan(lse[0, 0])
    rest = np.ones((new, 2), bool)
    rest[0, 0] = False
    assert np.isfinite(out[rest]).all() and np.isfinite(lse[rest]).all()
    k[32:64] = np.nan                                       # every score of one wave's step
    out, lse = _one_request(kind, q, k, v, new, splits)
    assert np.isnan(out).all() and np.isnan(lse).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("new", [1, 20])
def test_many_small_weights_add_up(kind, new):
    """One key far above 8000 others, each 2^-27 of it: together they are all of the result.  A weight is rounded by half a step of its type (float16: of
    2^-24 under a factor of 2^7, so 2^-32 of the largest), the result once, and two sums of 8000 terms in float32 add 2^-10."""
    n, dim = 8000, 64
    q, k, v = np.zeros((new, 1, dim)), np.zeros((n, 1, dim)), np.full((n, 1, dim), 64.0)
    q[:, 0, 0], k[7, 0, 0], v[7] = 1.0, 8.0 * 27 * np.log(2), 0.0
    k = ref.rounded(k, kind)
    out, lse = _one_request(kind, q, k, v, new)
    for r in range(new):
        seen = n - new + r + 1
        w = np.exp(-k[7, 0, 0] / 8.0)
        want = 64 * (seen - 1) * w / (1 + (seen - 1) * w)
        slack = (ref.EPS[kind] + (2.0 ** -32 / w if kind == "float16" else 0.0) + ref.EPS[kind] + 2.0 ** -9) * want
        assert (np.abs(out[r] - want) <= slack).all(), (r, out[r, 0, 0], want)
