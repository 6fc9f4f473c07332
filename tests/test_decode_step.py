"""The decoder-step operators as they are used: through library nodes and ``torch.compile(backend="docc")``, a step of a decoder that
grows its cache, captured and replayed, on other streams and from several threads."""
import math
import threading

import pytest
import torch
import torch.nn.functional as F

from docc_b200 import _lib, nodes as N, ops

gpu = pytest.mark.gpu


def settle():
    ops.sync()
    torch.cuda.synchronize()


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


# ---- nodes --------------------------------------------------------------------------------------------------------------------------
def test_nodes_carry_their_parameters_and_are_mapped():
    made = [N.RMSNormNode(eps=1e-5, has_residual=True, quantise=True, group=128), N.RoPENode(interleaved=True, mscale=1.5, inverse=True),
            N.RoPEAppendNode(interleaved=True), N.PagedAttentionNode(scale=0.5, softcap=30.0, window=7), N.TokenLogProbsNode(k=4, scale=2.0)]
    mapper = N.B200LibraryNodeMapper(with_transfers=False)
    for node in made:
        assert mapper.try_map(node)
        assert N.LibraryNodeDispatcherRegistry.instance().get_library_node_dispatcher(node.key()) is not None
        with pytest.raises(N.InvalidSDFGException):
            node.validate()  # no outputs named
        node.outputs = [f"o{i}" for i in range(len(node.output_connectors))]
        node.validate()
    assert made[0].output_connectors == ("Q", "C", "S") and N.RMSNormNode().output_connectors == ("Y",)
    assert made[0].to_json()["group"] == 128 and made[3].to_json()["softcap"] == 30.0 and made[4].to_json()["k"] == 4


class Decoder:
    """One pre-norm attention layer with rotary positions and a paged cache, and a vocabulary head, as a program of library nodes."""

    def __init__(self, dtype, d=128, heads=8, kv=2, head_dim=16, vocab=300, page=4, pages=40, layout="hsd"):
        self.heads, self.kv, self.head_dim, self.page = heads, kv, head_dim, page
        w = lambda *s, seed: normal(*s, seed=seed, dtype=dtype, scale=s[1] ** -0.5).cuda()
        self.wqkv, self.wo, self.wv = w((heads + 2 * kv) * head_dim, d, seed=1), w(d, heads * head_dim, seed=2), w(vocab, d, seed=3)
        self.g1, self.g2 = (1 + 0.1 * normal(d, seed=4)).cuda(), (1 + 0.1 * normal(d, seed=5)).cuda()
        shape = (pages, kv, page, head_dim) if layout == "hsd" else (pages, page, kv, head_dim)
        self.kc, self.vc = torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda")
        if layout != "hsd":
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        freq, self.mscale = ops.rope_frequencies(head_dim, scaling="yarn", factor=4, original_length=64)
        self.freq = torch.from_numpy(freq).cuda()

    def run(self, node, env, inputs, outputs):
        node.inputs, node.outputs = inputs, outputs
        N.B200LibraryNodeMapper(with_transfers=False).try_map(node)
        N.LibraryNodeDispatcherRegistry.instance().dispatch(node, env)

    def step(self, x, res, positions, slots, table, lengths, ids, k=3):
        """Hidden state and residual of the tokens -> (log-probabilities of ids, top ids, residual)."""
        env = dict(x=x, res=res, g1=self.g1, g2=self.g2, wqkv=self.wqkv, wo=self.wo, wv=self.wv, p=positions, f=self.freq, kc=self.kc, vc=self.vc,
                   slots=slots, table=table, n=lengths, ids=ids)
        self.run(N.RMSNormNode(has_residual=True), env, ["x", "g1", "res"], ["y", "s"])
        self.run(N.LinearNode(), env, ["y", "wqkv"], ["qkv"])
        h, kv, d = self.heads, self.kv, self.head_dim
        env["q"], env["k"], env["v"] = (t.unflatten(1, (-1, d)) for t in env["qkv"].split([h * d, kv * d, kv * d], dim=1))
        self.run(N.RoPEAppendNode(mscale=self.mscale), env, ["q", "k", "v", "p", "f", "kc", "vc", "slots"], ["qr"])
        self.run(N.PagedAttentionNode(), env, ["qr", "kc", "vc", "table", "n"], ["o"])
        env["o2"] = env["o"].flatten(1)
        self.run(N.LinearNode(), env, ["o2", "wo"], ["a"])
        self.run(N.RMSNormNode(has_residual=True), env, ["a", "g2", "s"], ["y2", "s2"])
        self.run(N.LinearNode(), env, ["y2", "wv"], ["logits"])
        self.run(N.TokenLogProbsNode(k=k), env, ["logits", "ids"], ["lp", "ent", "tids", "tlp"])
        return env["lp"], env["ent"], env["tids"], env["tlp"], env["s2"]

    def exact(self, xs, ress, ids):
        """The same for the last token of one sequence, from all its inputs, in fp64 on the host."""
        D = lambda t: t.double().cpu()
        s = D(xs) + D(ress)
        rms = lambda t, g: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * D(g)
        h, kv, d = self.heads, self.kv, self.head_dim
        q, k, v = (t.unflatten(1, (-1, d)) for t in (rms(s, self.g1) @ D(self.wqkv).T).split([h * d, kv * d, kv * d], dim=1))
        angle = torch.arange(len(xs)).double()[:, None] * D(self.freq)
        c, si = self.mscale * torch.cos(angle)[:, None], self.mscale * torch.sin(angle)[:, None]
        turn = lambda t: torch.cat([t[..., : d // 2] * c - t[..., d // 2 :] * si, t[..., d // 2 :] * c + t[..., : d // 2] * si], -1)
        q, k = turn(q)[-1], turn(k)
        p = torch.softmax(torch.einsum("hd,jhd->hj", q, k.repeat_interleave(h // kv, 1)) / math.sqrt(d), 1)
        o = torch.einsum("hj,jhd->hd", p, v.repeat_interleave(h // kv, 1)).flatten()
        s2 = s[-1] + o @ D(self.wo).T
        lp = torch.log_softmax(rms(s2, self.g2) @ D(self.wv).T, 0)
        return lp[ids], -(lp.exp() * lp).sum(), lp, s2


def batch_of(step, page, B, pages_per_seq, dtype, d=128):
    """Inputs of one step: sequence b starts at step b (before that its token is padding)."""
    x, res = normal(B, d, seed=100 + step, dtype=dtype), normal(B, d, seed=500 + step, dtype=dtype)
    pos = torch.tensor([step - b for b in range(B)])
    table = (torch.arange(B)[:, None] * pages_per_seq + torch.arange(pages_per_seq).flip(0)[None]).int()
    live = pos >= 0
    at = pos.clamp(min=0)
    slots = torch.where(live, table.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page, -1)
    return x, res, at, slots, table, torch.where(live, at + 1, 0).int()


@gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2), (torch.bfloat16, 5e-2)])
@pytest.mark.parametrize("layout", ["hsd", "shd"])
def test_a_decoder_grows_its_cache(rt, dtype, tol, layout):
    """Ten steps of three sequences that start one after the other. The tolerance is that of the chain's three products and norms in the
    type: norm-wise the stated 1e-4 for fp32, and of 16-bit types a handful of roundings (2^-11 or 2^-8 each) of every intermediate."""
    m = Decoder(dtype, layout=layout)
    B, steps = 3, 10
    history = []
    for step in range(steps):
        x, res, pos, slots, table, lengths = batch_of(step, m.page, B, 4, dtype)
        history.append((x, res))
        ids = torch.tensor([5, 17, 299])
        lp, ent, tids, tlp, s2 = m.step(x.cuda(), res.cuda(), pos.cuda(), slots.cuda(), table.cuda(), lengths.cuda(), ids.cuda())
        settle()
        for b in range(B):
            if step < b:
                continue
            xs, rs = torch.stack([h[0][b] for h in history[b:]]), torch.stack([h[1][b] for h in history[b:]])
            want, h, every, want_s2 = m.exact(xs, rs, ids[b])
            scale = every.abs().max()
            assert abs(lp[b].double().cpu() - want) <= tol * scale
            assert abs(ent[b].double().cpu() - h) <= tol * scale
            assert (s2[b].double().cpu() - want_s2).abs().max() <= tol * want_s2.abs().max()
            assert (tlp[b].double().cpu() - every[tids[b].cpu()]).abs().max() <= tol * scale


@gpu
def test_a_captured_step_follows_its_inputs(rt):
    """The step captured once and replayed with new inputs, lengths and slots gives what eager calls give, bit for bit."""
    dtype = torch.bfloat16
    eager, captured = Decoder(dtype), Decoder(dtype)
    static = [t.cuda() for t in batch_of(0, 4, 3, 4, dtype)]
    ids = torch.tensor([5, 17, 299]).cuda()
    captured.step(*static, ids)
    settle()
    captured.kc.zero_()
    captured.vc.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    ops.set_stream(side.cuda_stream)  # before the capture begins
    try:
        with torch.cuda.graph(graph, stream=side):
            outs = captured.step(*static, ids)
    finally:
        ops.set_stream(torch.cuda.current_stream().cuda_stream)
    for step in range(8):
        new = batch_of(step, 4, 3, 4, dtype)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = eager.step(*[n.cuda() for n in new], ids)
        settle()
        live = [b for b in range(3) if b <= step]
        for g, w in zip(outs, want):
            assert torch.equal(g[live], w[live])


def attention_case(B, lengths, heads, kv, dim, page, seed, dtype=torch.bfloat16):
    need = [-(-n // page) for n in lengths]
    kc, vc = normal(sum(need) + 1, kv, page, dim, seed=seed, dtype=dtype).cuda(), normal(sum(need) + 1, kv, page, dim, seed=seed + 1, dtype=dtype).cuda()
    table = torch.zeros(B, max(need), dtype=torch.int32)
    for b in range(B):
        table[b, : need[b]] = torch.arange(sum(need[:b]), sum(need[: b + 1]))
    return normal(B, heads, dim, seed=seed + 2, dtype=dtype).cuda(), kc, vc, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


@gpu
def test_two_captured_graphs_do_not_share_their_scratch(rt):
    cases = [attention_case(2, [4000, 3000], 8, 2, 64, 16, s) for s in (1, 50)]
    torch.cuda.synchronize()
    want = [ops.paged_attention(*c) for c in cases]
    settle()
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    try:
        for s, c in zip(streams, cases):
            g = torch.cuda.CUDAGraph()
            ops.set_stream(s.cuda_stream)
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.paged_attention(*c))
            graphs.append(g)
    finally:
        ops.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@gpu
def test_a_captured_call_without_scratch_is_refused(rt):
    q, kc, vc, table, lengths = attention_case(1, [100], 2, 1, 64, 16, 3)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    args = (ord("b"), 1, 2, 1, 64, 0.125, 0.0, 0, q.data_ptr(), None, kc.data_ptr(), None, vc.data_ptr(), None, kc.shape[0], 16, table.data_ptr(),
            table.shape[1], table.shape[1], lengths.data_ptr(), out.data_ptr(), None, None)
    fn = _lib.lib().docc_b200_paged_attention
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ops.set_stream(side.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=side):
            status = fn(*args, None, 0, 0)
            out.zero_()
    finally:
        ops.set_stream(torch.cuda.current_stream().cuda_stream)
    assert status == 1
    assert fn(*args, q.data_ptr(), 64, 0) == 1  # too small a workspace
    assert fn(*args, None, 0, 0) == 0
    settle()


@gpu
def test_calls_on_another_stream_are_ordered_on_it(rt):
    """Inputs made on a side stream, the calls routed to it, the result read there: nothing else is synchronised."""
    q, kc, vc, table, lengths = attention_case(3, [700, 20, 300], 4, 2, 64, 16, 7)
    x, g = normal(500, 2048, seed=1, dtype=torch.bfloat16).cuda(), torch.ones(2048, device="cuda")
    torch.cuda.synchronize()
    want, want_y = ops.paged_attention(q, kc, vc, table, lengths), ops.rmsnorm(x, g)
    settle()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.set_stream(side.cuda_stream)
        try:
            for _ in range(5):
                busy = torch.randn(4000, 4000, device="cuda")
                busy = busy @ busy
                q2, x2 = q * 1, x * 1  # queued behind the product
                got, y = ops.paged_attention(q2, kc, vc, table, lengths), ops.rmsnorm(x2, g)
                got2, y2 = got * 1, y * 1
        finally:
            ops.set_stream(torch.cuda.default_stream().cuda_stream)
    side.synchronize()
    assert torch.equal(got2, want) and torch.equal(y2, want_y)


@gpu
def test_calls_from_several_threads(rt):
    """Every thread has its own context, stream and scratch."""
    cases = [attention_case(2, [2500 + 300 * i, 900], 8, 2, 64, 16, 20 + 10 * i) for i in range(4)]
    torch.cuda.synchronize()
    want = [ops.paged_attention(*c) for c in cases]
    settle()
    wrong, errors = [], []

    def work(i):
        try:
            ops.init(0)  # a private stream of this thread's
            for _ in range(30):
                got = ops.paged_attention(*cases[i])
                ops.sync()
                if not torch.equal(got, want[i]):
                    wrong.append(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong


@gpu
def test_a_chain_of_launches_sees_what_the_one_before_wrote(rt):
    """Each launch may begin while the one before drains; fifty norms in a row, each reading the other's output, equal fifty apart."""
    x = normal(300, 1024, seed=4, dtype=torch.bfloat16).cuda()
    r = normal(300, 1024, seed=5, dtype=torch.bfloat16).cuda()
    g = (1 + 0.01 * normal(1024, seed=6)).cuda()
    a, ra = x, r
    for _ in range(50):
        a, ra = ops.rmsnorm(a, g, ra)
        torch.cuda.synchronize()
    b, rb = x, r
    for _ in range(50):
        b, rb = ops.rmsnorm(b, g, rb)
    settle()
    assert torch.equal(a, b) and torch.equal(ra, rb)


# ---- the compiled host side -----------------------------------------------------------------------------------------------------------
def test_the_compiled_calls_answer_none_to_what_they_do_not_take():
    module = ops._compiled(torch.zeros(1))
    assert module and module is ops._native
    x = torch.zeros(2, 3)
    for name, count in (("rmsnorm", 4), ("rmsnorm_quant", 5), ("rope", 7), ("rope_append", 11), ("paged_attention", 10), ("token_logprobs", 4)):
        fn = getattr(module, name)
        assert fn() is None and fn(*[None] * count) is None and fn(*[x] * count) is None and fn(*["a"] * count) is None
        assert fn(*[x.numpy()] * count) is None and fn(*[1.5] * (count + 3)) is None


def both_ways(monkeypatch, call):
    """The call through the compiled host side, with proof that it took it, and through the Python one."""
    taken = []

    class Spy:
        def __getattr__(self, name):
            def fn(*args):
                got = getattr(module, name)(*args)
                taken.append(got is not None)
                return got

            return fn

    module = ops._compiled(torch.zeros(1))
    monkeypatch.setattr(ops, "_native", Spy())
    compiled = call()
    settle()
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.setattr(ops, "_compiled", lambda x: False)
    plain = call()
    settle()
    monkeypatch.undo()
    assert taken == [True]
    compiled, plain = (r if isinstance(r, tuple) else (r,) for r in (compiled, plain))
    assert len(compiled) == len(plain)
    for a, b in zip(compiled, plain):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.device == b.device and not a.requires_grad
        torch.testing.assert_close(a.float(), b.float(), rtol=0, atol=0, equal_nan=True)  # NaN: the id that is no token


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_both_host_sides_make_the_same_call(rt, monkeypatch, dtype):
    wide = normal(6, 1000, seed=1, dtype=dtype).cuda()
    x, r, g = wide[:, :256], wide[:, 256:512], torch.nn.Parameter(normal(256, seed=2).cuda())
    both_ways(monkeypatch, lambda: ops.rmsnorm(x, g, r))
    both_ways(monkeypatch, lambda: ops.rmsnorm(x.contiguous().view(2, 3, 256)))
    both_ways(monkeypatch, lambda: ops.rmsnorm_quant(x, g, r, group=128))
    both_ways(monkeypatch, lambda: ops.rmsnorm_quant(x.contiguous().view(2, 3, 256), group=0, eps=1e-5))
    q, k, v = (t.unflatten(1, (-1, 32)) for t in wide[:, : 32 * 12].split([256, 64, 64], dim=1))
    pos, freq = torch.arange(6).cuda(), torch.from_numpy(ops.rope_frequencies(32)[0]).cuda()
    both_ways(monkeypatch, lambda: ops.rope(q, pos, freq, interleaved=True, mscale=2))
    both_ways(monkeypatch, lambda: ops.rope(q, pos, freq, inverse=True, out=torch.empty(6, 16, 32, dtype=dtype, device="cuda")[:, ::2]))
    slots = torch.tensor([3, 9, -1, 0, 15, 7]).cuda()
    kc, vc = normal(4, 2, 4, 32, seed=5, dtype=dtype).cuda(), normal(4, 4, 2, 32, seed=6, dtype=dtype).cuda().transpose(1, 2)
    both_ways(monkeypatch, lambda: (ops.rope_append(q, k, v, pos, freq, kc, vc, slots), kc.clone(), vc.contiguous()))
    table, lengths = torch.arange(4).int().cuda().view(2, 2), torch.tensor([7, 5], dtype=torch.int32).cuda()
    both_ways(monkeypatch, lambda: ops.paged_attention(q[:2], kc, vc, table, lengths, return_lse=True))
    both_ways(monkeypatch, lambda: ops.paged_attention(q[:2].contiguous(), kc, vc, table, lengths, scale=0.3, softcap=4, window=3))
    ids = torch.tensor([0, 5, 999, -1, 4, 2]).cuda()
    both_ways(monkeypatch, lambda: ops.token_logprobs(wide, ids)[:2])
    both_ways(monkeypatch, lambda: ops.token_logprobs(wide[:, :700], ids, k=4, scale=0.5))


# ---- torch.compile ------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("eps", [None, 1e-5])
def test_rms_norm_through_torch_compile(rt, dtype, tol, eps):
    from docc_b200 import torch as dt

    torch._dynamo.reset()
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.RMSNorm(96, eps=eps), torch.nn.Linear(96, 8)).cuda().to(dtype)
    x = (1e-2 * torch.randn(5, 64)).to(dtype).cuda()
    with torch.no_grad():
        dt.set_backend_options(target="cuda")
        try:
            got = torch.compile(model, backend="docc")(x)
        finally:
            dt.set_backend_options()
        settle()
        h = F.linear(x.double(), model[0].weight.double(), model[0].bias.double())
        e = torch.finfo(torch.float32).eps if eps is None else eps  # what torch adds, whatever the type
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + e) * model[1].weight.double()
        want = F.linear(h, model[2].weight.double(), model[2].bias.double())
    assert (got.double() - want).abs().max() <= tol * want.abs().max()


def test_rms_norm_that_has_no_node_is_refused():
    from docc_b200 import torch as dt

    with pytest.raises(dt.UnsupportedGraph):
        dt._rms_norm(torch.zeros(2, 3, 4), (3, 4))
    with pytest.raises(dt.UnsupportedGraph):
        dt._rms_norm(torch.zeros(2, 4, dtype=torch.float64), (4,))
