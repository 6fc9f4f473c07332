"""Edges of the decoding-step operators that their other tests do not reach: values at the middle between two 8-bit codes, one key far
above all others, visible infinities, rows around the shared memory that needs no opt-in, a failing call's status, and a host side that
could not be built."""
import ctypes
import math
import os
import subprocess
import sys
import threading
import time
import warnings

import numpy as np
import pytest
import torch

from docc_b200 import _lib, build, ops
from test_decode_ops import DTYPES, E, TINY, U, attention_exact, close, gpu, normal, paged_problem, rms_exact, rms_tolerance, settle

# ---- 8-bit codes ------------------------------------------------------------------------------------------------------------------
def e4m3_middles():
    """The values half way between two neighbouring codes, from the smallest on."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return (codes[1:] + codes[:-1]) / 2


def codes_problem(cols, tops, seed):
    """gamma whose quotients by its groups' scales lie at the middles between two codes and up to three steps of fp32 beside them.
    Signs as an input have a mean square of exactly 1, so the norm is the signed gamma, bit for bit."""
    rng = np.random.default_rng(seed)
    width = -(-cols // len(tops))
    gamma = np.zeros(cols, dtype=np.float32)
    for i, top in enumerate(np.float32(tops)):
        part = gamma[i * width : (i + 1) * width]
        scale = top / np.float32(448)
        y = (scale.astype(np.float64) * rng.choice(e4m3_middles().numpy(), len(part))).astype(np.float32)
        for _ in range(3):
            y = np.where(rng.random(len(part)) < 0.4, np.nextafter(y, np.float32(rng.choice([0, 1e38]))), y)
        part[:] = np.minimum(y, top)
        part[0] = top
    return torch.from_numpy(gamma)


def codes_of(y, group):
    """scale = max|y| / 448 and e4m3(y / scale), each rounded once from fp32 operands; a scale of 0 has codes of 0."""
    scales, codes = [], []
    for part in y.split(y.shape[1] if group == 0 else 128, dim=1):
        scale = part.abs().amax(1, keepdim=True) / 448
        q = torch.where(scale > 0, part / scale, 0.0).clamp(-448, 448)
        scales.append(scale)
        codes.append(q.to(torch.float8_e4m3fn))
    return torch.cat([c.view(torch.uint8) for c in codes], 1), torch.cat(scales, 1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("rows,cols", [(3, 256), (5, 1024), (2, 4096), (2, 8192), (3, 257), (4, 1001), (2, 5003), (1300, 333), (1200, 1022)])
def test_codes_are_those_of_the_quotient(rt, rows, cols, group, dtype):
    """Bit for bit where y / scale lies at the middle between two codes or a step beside it: the quotient decides, not a product with a
    rounded reciprocal."""
    tops = [1.7] if group == 0 else [1.7 + 0.37 * i for i in range(-(-cols // 128))]
    gamma = codes_problem(cols, tops, seed=rows + cols)
    x = torch.where(normal(rows, cols, seed=cols) < 0, -1.0, 1.0)
    q, scales = ops.rmsnorm_quant(x.to(dtype).cuda(), gamma.cuda(), eps=0.0, group=group)
    settle()
    want, want_scales = codes_of(x * gamma, group)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(q.cpu().view(torch.uint8), want)


@gpu
@pytest.mark.parametrize("cols", [1024, 1021])
def test_codes_under_tiny_scales(rt, cols):
    """Scales below fp32's smallest normal number, whose own rounding is large, one that rounds to zero, and a group of zeros."""
    tops = [1.5, 3e-30, 1e-38, 448 * 2.0**-140, 5 * 2.0**-141, 2.0**-149, 0.0, 1e-42]
    gamma = codes_problem(cols, tops, seed=cols)
    x = torch.where(normal(3, cols, seed=1) < 0, -1.0, 1.0)
    q, scales = ops.rmsnorm_quant(x.cuda(), gamma.cuda(), eps=0.0, group=128)
    settle()
    want, want_scales = codes_of(x * gamma, 128)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(q.cpu().float(), want.view(torch.float8_e4m3fn).float())  # -0 and 0 are one value
# ---- attention: one key far above the others --------------------------------------------------------------------------------------
def sink_problem(B, length, gap, group, kv, dim, dtype, page=16, seed=0):
    """Sequences that share their pages: the first key scores ``gap`` above the others, which lie around 0, and its value is zero."""
    pages = -(-length // page)
    kc, vc = torch.zeros(pages, kv, page, dim, dtype=dtype), 1 + 0.1 * normal(pages, kv, page, dim, seed=seed).to(dtype)
    kc[..., 0] = (0.1 * normal(pages, kv, page, seed=seed + 1)).to(dtype)
    kc[0, :, 0, 0] = gap
    vc[0, :, 0] = 0
    q = torch.zeros(1, group * kv, dim, dtype=dtype)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32)[None]
    lengths = torch.tensor([length], dtype=torch.int32)
    got = ops.paged_attention(q.expand(B, -1, -1).contiguous().cuda(), kc.cuda(), vc.cuda(), table.expand(B, -1).contiguous().cuda(),
                              lengths.expand(B).contiguous().cuda(), scale=1.0, return_lse=True)
    settle()
    want = attention_exact(q, kc, vc, table, lengths, 1.0, 0.0, 0)
    for g, w, tol in ((got[0], want[0], want[1]), (got[1], want[2], want[3])):
        close(g, w.expand(g.shape), tol.expand(g.shape))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [16.0, 17.5, 20.0, 24.0])
@pytest.mark.parametrize("whole", [True, False])
def test_attention_keeps_small_probabilities(rt, whole, gap, dtype):
    """Thousands of keys whose probabilities, each below the smallest number of fp16, make up the whole output: a row per block, and one
    row split over all blocks."""
    blocks = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    sink_problem(blocks if whole else 1, 8192, gap, 1, 1, 64, dtype)


@gpu
@pytest.mark.parametrize("group,kv,dim", [(4, 2, 80), (16, 1, 128), (12, 2, 64), (2, 1, 256), (20, 1, 96)])
def test_attention_keeps_small_probabilities_in_every_kernel(rt, group, kv, dim):
    sink_problem(3, 3000, 19.0, group, kv, dim, torch.float16, seed=5)
# ---- attention: infinities that are seen ------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads", [([1, 2, 40, 700], 4), ([5000, 33], 16)])
def test_attention_of_a_visible_infinite_value(rt, lengths, heads, dtype):
    """p inf = inf for every p > 0, in its own column only; two of opposite sign, or a NaN, give a NaN."""
    q, kc, vc, table, lengths = paged_problem(lengths, heads, 1, 64, 16, dtype)
    settle()
    plain = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    settle()
    bad = {5: [math.inf], 9: [-math.inf], 20: [math.inf, -math.inf], 31: [math.nan]}
    want = plain.clone()
    for b, n in enumerate(lengths.tolist()):
        for column, values in bad.items():
            if len(values) > n:
                continue
            for i, v in enumerate(values):
                j = (n - 1 - 7 * i) % n
                vc[int(table[b, j // 16]), 0, j % 16, column] = v
            want[b, :, column] = sum(values)
    settle()
    got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    settle()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, 1e4, -1e4), want.nan_to_num(0.0, 1e4, -1e4))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_an_infinite_value_of_small_probability(rt, dtype):
    """A key far below the one that dominates still has a probability, and so an infinite share."""
    gap = 26.0 if dtype == torch.float16 else 85.0  # e^-26 = 2^-37.5, e^-85 = 2^-122.6
    kc, vc = torch.zeros(1, 1, 16, 64, dtype=dtype, device="cuda"), torch.ones(1, 1, 16, 64, dtype=dtype, device="cuda")
    kc[0, 0, 3, 0], vc[0, 0, 7, 2] = gap, math.inf
    q = torch.zeros(1, 2, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1
    settle()
    got = ops.paged_attention(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([16], dtype=torch.int32).cuda(), scale=1.0)
    settle()
    assert (got[..., 2] == math.inf).all() and (got[..., :2] == 1).all() and (got[..., 3:] == 1).all()
# ---- RMS norm: rows around the 48 KB of shared memory that need no opt-in ---------------------------------------------------------
def norm_of_width(cols, dtype, quant, offset=0, rows=2):
    flat = normal(rows * cols + offset, seed=cols, dtype=dtype)
    x = flat[offset:].view(rows, cols)
    on_device = flat.cuda()[offset:].view(rows, cols)
    if quant:
        q, scales = ops.rmsnorm_quant(on_device, eps=1e-6)
        ops.sync()
        got = q.float().double().cpu() * scales.double().cpu()
        _, y = rms_exact(x, None, None, 1e-6)
        drift = (cols / 32 + 20) * E
        close(got, y, y.abs() * (2.0**-4 + 4 * drift) + y.abs().amax(1, keepdim=True) / 448 * 2.0**-10 * (1 + 4 * drift))
    else:
        got = ops.rmsnorm(on_device, eps=1e-6)
        ops.sync()
        _, y = rms_exact(x, None, None, 1e-6)
        close(got, y, y.abs() * U[dtype] * 1.01 + rms_tolerance(y, cols) + TINY[dtype])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant", [False, True])
def test_rmsnorm_of_widths_beside_48_kb(rt, quant, dtype):
    for cols, offset in ((12281, 0), (12287, 0), (12288, 1), (12289, 0), (32767, 0), (12283, 0)):
        norm_of_width(cols, dtype, quant, offset)


@gpu
def test_rmsnorm_of_such_a_width_is_the_first_call(rt):
    """In a process of its own, where no wider row has been seen before."""
    code = ("import torch, test_decode_edges as t; from docc_b200 import ops; ops.init(0); "
            "ops.set_stream(torch.cuda.current_stream().cuda_stream); "
            "[t.norm_of_width(12281, d, q) for d in t.DTYPES for q in (False, True)]; print('done')")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(__file__), os.path.dirname(os.path.dirname(__file__))]))
    got = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "done" in got.stdout, got.stderr[-2000:]


@gpu
def test_rmsnorm_of_two_widths_from_two_threads(rt):
    """Neither thread's rows change what the other's kernel may use."""
    xs = [normal(2, cols, seed=cols, dtype=torch.bfloat16).cuda() for cols in (12301, 32767)]
    torch.cuda.synchronize()
    want = [ops.rmsnorm(x) for x in xs]
    settle()
    wrong = []

    def work(i):
        try:
            ops.init(0)
            for _ in range(300):
                got = ops.rmsnorm(xs[i])
                ops.sync()
                if not torch.equal(got, want[i]):
                    wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
# ---- the compiled host side: statuses ---------------------------------------------------------------------------------------------
def ordinary_calls():
    """A call of every entry that the compiled host side takes."""
    x, pos, freq = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(32, dtype=torch.float64, device="cuda")
    cache, table, lengths = torch.zeros(3, 4, 16, 64, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    return {"docc_b200_rmsnorm": lambda: ops.rmsnorm(x), "docc_b200_rmsnorm_q8": lambda: ops.rmsnorm_quant(x),
            "docc_b200_rope": lambda: ops.rope(x, pos, freq, out=x),
            "docc_b200_rope_append": lambda: ops.rope_append(x, x, x, pos, freq, cache, cache, pos, out=x),
            "docc_b200_paged_attention": lambda: ops.paged_attention(x, cache, cache, table, lengths),
            "docc_b200_token_logprobs": lambda: ops.token_logprobs(x[:, 0], pos, k=2)}


def bound_to(entries):
    """Binds the compiled host side to ``entries`` where given, to the library's own otherwise."""
    module = ops._compiled(torch.zeros(1))
    address = lambda name: ctypes.cast(entries.get(name, getattr(_lib.lib(), name)), ctypes.c_void_p).value
    module.bind(*(address(name) for name in ops._NATIVE), _lib.check)


@gpu
@pytest.mark.parametrize("name", ["docc_b200_rmsnorm", "docc_b200_rmsnorm_q8", "docc_b200_rope", "docc_b200_rope_append", "docc_b200_paged_attention",
                                  "docc_b200_token_logprobs"])
def test_a_call_that_failed_is_not_made_again(rt, name):
    """A status that may come after the kernel was queued raises from the one call; rotated in place, a second one would turn twice."""
    restype, argtypes = _lib.SIGNATURES[name]
    calls = []
    entry = ctypes.CFUNCTYPE(restype, *argtypes)(lambda *args: calls.append(args) or status)
    run = ordinary_calls()[name]
    rt.docc_b200_launch_count(1)
    try:
        bound_to({name: entry})
        for status in (3, 4, 5, 6):  # CUDA, out of memory, no device, timeout
            calls.clear()
            with pytest.raises(_lib.DoccB200Error) as e:
                run()
            assert e.value.status == status and name in str(e.value) and len(calls) == 1
        assert rt.docc_b200_launch_count(0) == 0
        for status in (1, 2):  # refused before anything was queued: the Python side makes the call, and here it succeeds
            calls.clear()
            run()
            assert len(calls) == 1
        assert rt.docc_b200_launch_count(0) >= 2
    finally:
        bound_to({})
    settle()
@gpu
def test_other_threads_run_while_an_entry_waits(rt):
    """The entry stands for one that waits for a stream: the C library's poll(fds, 0, cols), which sleeps ``cols`` milliseconds and
    returns 0, in the place of rmsnorm(prec, 0 rows, cols, ...)."""
    x = torch.empty(0, 400, device="cuda")
    stop, ticks = threading.Event(), []

    def tick():
        while not stop.wait(0.002):
            ticks.append(time.monotonic())

    thread = threading.Thread(target=tick)
    try:
        bound_to({"docc_b200_rmsnorm": ctypes.CDLL(None).poll})
        thread.start()
        begin = time.monotonic()
        ops.rmsnorm(x)
        end = time.monotonic()
    finally:
        bound_to({})
        stop.set()
        thread.join()
    assert end - begin >= 0.39 and len([t for t in ticks if begin < t < end]) >= 20
# ---- the compiled host side: where it cannot be built -----------------------------------------------------------------------------
@pytest.mark.parametrize("compiler", ["false", "/no/such/compiler"])
def test_the_runtime_is_built_where_the_host_side_cannot_be(monkeypatch, tmp_path, compiler):
    """A box with torch but without its compiler or the interpreter's headers; what an earlier build left there is not kept."""
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(build, "_build_runtime", lambda verbose: None)
    monkeypatch.setenv("CXX", compiler)
    with open(build.host_path(), "w") as fh:
        fh.write("built by another compiler")
    with pytest.warns(RuntimeWarning, match="could not be compiled"):
        assert build.build() == build.LIB_PATH
    assert not os.path.exists(build.host_path()) and not build.host_is_current()


def test_the_host_side_belongs_to_one_torch_and_interpreter(monkeypatch):
    here = build.host_path()
    assert build.host_is_current() and os.path.exists(here)
    with monkeypatch.context() as m:
        m.setattr(build, "_torch_version", lambda: "0.1")
        assert build.host_path() != here and not build.host_is_current()
    with monkeypatch.context() as m:
        m.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-999")
        assert build.host_path() != here and not build.host_is_current()
    with monkeypatch.context() as m:
        m.setattr(build, "_torch_root", lambda: None)  # no torch, no host side
        assert build.host_path() is None and build.host_is_current()


def test_calls_without_the_compiled_host_side(monkeypatch):
    """They take the Python path, which says what is wrong, and warn once."""
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.setattr(build, "_torch_version", lambda: "0.1")
    with pytest.warns(RuntimeWarning, match="cannot be loaded"):
        with pytest.raises(TypeError, match="CUDA device"):
            ops.rmsnorm(torch.zeros(2, 8))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(TypeError, match="CUDA device"):
            ops.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


@gpu
def test_results_without_the_compiled_host_side(rt, monkeypatch):
    x = normal(5, 300, seed=1).cuda()
    want = ops.rmsnorm(x)
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.setattr(build, "_torch_version", lambda: "0.1")
    with pytest.warns(RuntimeWarning, match="cannot be loaded"):
        got = ops.rmsnorm(x)
    settle()
    assert torch.equal(got, want)
# ---- scratch ----------------------------------------------------------------------------------------------------------------------
@gpu
def test_the_cache_attention_leaves_the_scratch_of_a_captured_attention_alone(rt):
    """fp32 attention over contiguous keys may be captured with the thread's scratch; an eager call over the cache that needs more than
    that must neither use the same memory nor give it back."""
    changed = []

    def work():  # a new thread has scratch of its own, which begins empty
        try:
            ops.init(0)
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            ops.set_stream(stream.cuda_stream)
            with torch.cuda.stream(stream):
                q = normal(1, 2, 256, 64, seed=1).cuda()
                want = ops.attention(q, q, q)
                with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
                    got = ops.attention(q, q, q)
                paged = paged_problem([3000], 16, 1, 128, 16, torch.bfloat16)
                out = ops.paged_attention(paged[0].cuda(), paged[1], paged[2], paged[3].cuda(), paged[4].cuda())
                held = [ops.DeviceArray.from_numpy(np.full(100_000, 7, dtype=np.float32)) for _ in range(8)]
                graph.replay()
                stream.synchronize()
                changed.extend(i for i, h in enumerate(held) if not (h.to_numpy() == 7).all())
                changed.extend([] if torch.equal(got, want) and torch.isfinite(out).all() else ["result"])
            ops.sync()
        except Exception as e:  # noqa: BLE001
            changed.append(e)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert not changed
# ---- outputs of calls without elements --------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_of_rows_of_nothing(rt, dtype):
    """One scale per row is a row's even if it has no columns: zero, like that of a row of zeros."""
    for _ in range(4):
        used = torch.full((5, 1), 7.0, device="cuda")
        settle()
        del used  # the next allocation of this size is likely to hold sevens
        q, scales = ops.rmsnorm_quant(torch.empty(5, 0, dtype=dtype, device="cuda"), group=0)
        settle()
        assert q.shape == (5, 0) and scales.shape == (5, 1) and (scales == 0).all()
    assert ops.rmsnorm_quant(torch.empty(5, 0, dtype=dtype, device="cuda"), group=128)[1].shape == (5, 0)
    assert (ops.rmsnorm_quant(np.empty((5, 0), dtype=np.float32))[1] == 0).all()
@gpu
def test_attention_of_heads_without_elements_has_no_lse(rt):
    """Its scores would be those of empty products; the call that would have to return them is refused."""
    q, cache = torch.empty(2, 4, 0, device="cuda"), torch.empty(3, 2, 16, 0, device="cuda")
    table, lengths = torch.zeros(2, 1, dtype=torch.int32).cuda(), torch.ones(2, dtype=torch.int32).cuda()
    assert ops.paged_attention(q, cache, cache, table, lengths).shape == (2, 4, 0)
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.paged_attention(q, cache, cache, table, lengths, return_lse=True)
    assert e.value.status == 1
    settle()
# ---- arrays of the runtime's own pool ---------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_calls_on_arrays_of_the_pool(rt, dtype):
    """A whole step on DeviceArrays gives DeviceArrays that hold what torch tensors give."""
    held = lambda t: ops.DeviceArray.from_numpy(t.cpu().numpy())
    same = lambda a, t: isinstance(a, ops.DeviceArray) and np.array_equal(a.to_numpy(), t.cpu().numpy())
    x, gamma, res = normal(4, 256, seed=1, dtype=dtype).cuda(), 1 + 0.1 * normal(256, seed=2).cuda(), normal(4, 256, seed=3, dtype=dtype).cuda()
    both = [(ops.rmsnorm(held(x), held(gamma)),), (ops.rmsnorm(x, gamma),)]
    both[0] += ops.rmsnorm(held(x), held(gamma), held(res))
    both[1] += ops.rmsnorm(x, gamma, res)
    codes = ops.rmsnorm_quant(held(x), held(gamma), held(res), group=128)
    want = ops.rmsnorm_quant(x, gamma, res, group=128)
    both[0] += codes
    both[1] += (want[0].view(torch.uint8), *want[1:])
    q, k, v = normal(4, 8, 64, seed=4, dtype=dtype).cuda(), normal(4, 2, 64, seed=5, dtype=dtype).cuda(), normal(4, 2, 64, seed=6, dtype=dtype).cuda()
    pos, freq = torch.arange(4).cuda() + 900, torch.from_numpy(ops.rope_frequencies(32)[0]).cuda()
    kc, vc, slots = torch.zeros(3, 2, 16, 64, dtype=dtype).cuda(), torch.zeros(3, 2, 16, 64, dtype=dtype).cuda(), torch.tensor([0, 17, 18, -1]).cuda()
    table, lengths = torch.tensor([[0, 1], [1, 0], [1, 2], [2, 0]], dtype=torch.int32).cuda(), torch.tensor([20, 3, 5, 0], dtype=torch.int32).cuda()
    both[0] += (ops.rope(held(q), held(pos), held(freq), interleaved=True, mscale=1.5),)
    both[1] += (ops.rope(q, pos, freq, interleaved=True, mscale=1.5),)
    dk, dv = held(kc), held(vc)
    both[0] += (ops.rope_append(held(q), held(k), held(v), held(pos), held(freq), dk, dv, held(slots)), dk, dv)
    both[1] += (ops.rope_append(q, k, v, pos, freq, kc, vc, slots), kc, vc)
    settle()
    both[0] += ops.paged_attention(held(q), dk, dv, held(table), held(lengths), window=9, return_lse=True)
    both[1] += ops.paged_attention(q, kc, vc, table, lengths, window=9, return_lse=True)
    ids = torch.tensor([0, 255, 3, -1]).cuda()
    got, want = ops.token_logprobs(held(x), held(ids), k=4), ops.token_logprobs(x, ids, k=4)
    settle()
    for a, t in zip(*both):
        assert same(a, t)
    for a, t in zip(got, want):
        assert isinstance(a, ops.DeviceArray) and np.array_equal(a.to_numpy(), t.cpu().numpy(), equal_nan=a.dtype.kind == "f")
@gpu
def test_an_entry_keeps_the_memory_of_its_arguments(rt):
    """Another thread may run while the entry does. What it takes from an argument meanwhile (here the entry itself does) is not handed
    out again before the entry has returned."""
    restype, argtypes = _lib.SIGNATURES["docc_b200_rmsnorm"]
    x, before, after = torch.zeros(37, 1024, device="cuda"), [], []
    settle()

    def entry(*args):
        before.append(x.data_ptr())
        x.set_()
        after.append(torch.empty(37, 1024, device="cuda").data_ptr())
        return 0

    try:
        stand_in = ctypes.CFUNCTYPE(restype, *argtypes)(entry)
        bound_to({"docc_b200_rmsnorm": stand_in})
        ops.rmsnorm(x)
    finally:
        bound_to({})
    assert len(before) == len(after) == 1 and before != after
