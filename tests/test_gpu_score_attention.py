"""GPU tests of the score-modified attention (prompt form, gradients, single-token form, shared prefix) against the
64-bit reference in oracle/score_attention.py, whose error bounds are the tolerances."""
import ctypes

import pytest
import torch

from oracle import score_attention as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def no_wait_ran_out(binding):
    yield
    st = ctypes.c_uint(1)
    torch.cuda.synchronize()
    assert binding.load_library().sm120_get_kernel_status(0, ctypes.byref(st), 1) == 0 and st.value == 0


def normal(gen, *shape, dtype, factor=1.0, layout="bhsd"):
    if layout == "bshd" and len(shape) == 4:
        return (torch.randn((shape[0], shape[2], shape[1], shape[3]), generator=gen, device="cuda") * factor).to(dtype).transpose(1, 2)
    return (torch.randn(shape, generator=gen, device="cuda") * factor).to(dtype)


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    same = torch.isneginf(want) & torch.isneginf(got)
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).nan_to_num(1e30).max()):.3g} x its bound at " \
                          f"{[int(x) for x in torch.nonzero(bad)[0]]}"


def offsets(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def masks(kind, b, sq, sk):
    """Options of the call and the reference's visible keys."""
    opt = {}
    if kind in ("causal", "prefix", "documents_causal"):
        opt["causal_mask"] = True
    if kind == "prefix":
        opt["prefix_lengths"] = offsets([(sk // 3 + 7 * e) if e % 2 == 0 else 0 for e in range(b)])
    if "documents" in kind:
        # ragged documents, an empty one, padding in front (odd entries) and behind
        opt["document_offsets"] = offsets([[e % 2 * (sk // 9), sk // 4, sk // 4, sk // 2 + 3 * e, max(sk // 2 + 3 * e, sk - sk // 10)] for e in range(b)]).clamp(max=sk)
    seen = ref.visible(b, sq, sk, causal="causal_mask" in opt, prefix_lengths=opt.get("prefix_lengths"),
                       document_offsets=opt.get("document_offsets"), device="cuda")
    return opt, seen


def train_and_check(ops, gen, dtype, b, h, hk, sq, sk, d, kind, softcap=None, alibi=False, layout="bhsd", scale=None, factor=1.0, grads=True):
    q, do = (normal(gen, b, h, sq, d, dtype=dtype, layout=layout, factor=f) for f in (factor, 1.0))
    k, v = (normal(gen, b, hk, sk, d, dtype=dtype, layout=layout) for _ in range(2))
    opt, seen = masks(kind, b, sq, sk)
    slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if alibi else None
    opt.update(softcap=softcap, alibi_slopes=slopes, scale=scale)
    out, lse = ops.score_attention(q, k, v, return_lse=True, **opt)
    what = (str(dtype), b, h, hk, sq, sk, d, kind, softcap, alibi, layout)
    want = ref.attention(q, k, v, scale=scale, softcap=softcap, slopes=slopes, seen=seen, grad_out=do if grads else None)
    within(out, want["out"], want["out_tol"], ("out", *what))
    within(lse, want["lse"], want["lse_tol"], ("lse", *what))
    assert torch.equal(ops.score_attention(q, k, v, **opt), out), what            # the same with and without lse
    if grads:
        got = ops.score_attention_grad(do, q, k, v, out, lse, **opt)
        for name, g in zip(("dq", "dk", "dv"), got):
            within(g, want[name], want[name + "_tol"], (name, *what))
        again = ops.score_attention_grad(do, q, k, v, out, lse, **opt)
        assert all(torch.equal(x, y) for x, y in zip(got, again)), what            # a fixed order of summation


SEQUENCES = [
    # b, h, hk, sq, sk, d, mask, softcap, alibi, layout
    (1, 1, 1, 1, 1, 64, "full", None, False, "bhsd"),
    (1, 2, 1, 1, 1, 128, "causal", None, True, "bhsd"),
    (2, 2, 2, 1, 300, 64, "causal", 20.0, True, "bhsd"),
    (1, 2, 2, 128, 128, 128, "full", None, False, "bhsd"),
    (2, 4, 2, 127, 129, 64, "causal", None, False, "bshd"),
    (1, 2, 1, 257, 257, 128, "causal", None, False, "bhsd"),
    (1, 2, 1, 257, 257, 128, "causal", 30.0, True, "bshd"),
    (2, 6, 2, 200, 333, 80, "causal", None, True, "bhsd"),
    (2, 3, 1, 333, 200, 96, "causal", 20.0, False, "bshd"),          # more queries than keys: rows that see nothing
    (3, 2, 2, 300, 300, 64, "prefix", None, False, "bhsd"),
    (2, 2, 2, 515, 700, 128, "prefix", 25.0, True, "bshd"),
    (2, 4, 4, 500, 500, 64, "documents", None, False, "bhsd"),
    (3, 4, 2, 700, 700, 128, "documents_causal", None, True, "bhsd"),
    (2, 2, 1, 400, 640, 128, "documents", 15.0, True, "bshd"),
    (2, 2, 1, 300, 900, 64, "documents_causal", None, False, "bshd"),
    (1, 8, 1, 1030, 1030, 128, "full", None, True, "bhsd"),
    (1, 2, 2, 1200, 1200, 8, "causal", None, True, "bhsd"),
    (1, 2, 2, 100, 2500, 120, "full", 50.0, False, "bhsd"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", SEQUENCES, ids=lambda c: "-".join(map(str, c)))
def test_sequences(ops, dtype, case):
    b, h, hk, sq, sk, d, kind, softcap, alibi, layout = case
    gen = torch.Generator(device="cuda").manual_seed(100 + sq + sk)
    train_and_check(ops, gen, DT[dtype], b, h, hk, sq, sk, d, kind, softcap, alibi, layout, factor=3.0 if softcap else 1.0)


@pytest.mark.parametrize("case", [SEQUENCES[i] for i in (1, 2, 6, 8, 10, 13)] + [(1, 2, 2, 70, 90, 33, "causal", 20.0, True, "bhsd"),
                                                                                 (1, 2, 1, 40, 50, 256, "full", None, True, "bshd")],
                         ids=lambda c: "-".join(map(str, c)))
def test_sequences_float32(ops, case):
    b, h, hk, sq, sk, d, kind, softcap, alibi, layout = case
    gen = torch.Generator(device="cuda").manual_seed(7)
    train_and_check(ops, gen, torch.float32, b, h, hk, sq, sk, d, kind, softcap, alibi, layout, factor=3.0 if softcap else 1.0)


@pytest.mark.parametrize("d", [5, 33, 136, 200, 256])
def test_head_dims_off_the_tensor_core_path(ops, d):
    gen = torch.Generator(device="cuda").manual_seed(d)
    train_and_check(ops, gen, torch.bfloat16, 1, 2, 1, 65, 130, d, "causal", 20.0, True)


def test_seeded_sweep(ops):
    import random
    r = random.Random(11)
    gen = torch.Generator(device="cuda").manual_seed(11)
    for _ in range(30):
        hk, g = r.choice([1, 2, 3]), r.choice([1, 2, 4])
        sq = r.choice([1, r.randint(2, 64), r.randint(65, 700)])
        sk = sq + r.choice([0, 0, r.randint(1, 400)])
        train_and_check(ops, gen, r.choice([torch.bfloat16, torch.float16]), r.randint(1, 3), hk * g, hk, sq, sk, r.choice([64, 128, 72, 96]),
                        r.choice(["full", "causal", "prefix", "documents", "documents_causal"]), r.choice([None, 20.0]), r.random() < 0.5,
                        r.choice(["bhsd", "bshd"]))


@pytest.mark.parametrize("scale", [1.0, -0.5, 0.0])
def test_large_growing_and_negative_scores(ops, scale):
    """Scores that grow from key tile to key tile move the running maximum again and again; a negative scale makes the smallest
    product the largest score; capped scores saturate."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    b, h, s, d = 1, 2, 900, 64
    q, do = normal(gen, b, h, s, d, dtype=torch.bfloat16), normal(gen, b, h, s, d, dtype=torch.bfloat16)
    grow = (1 + 0.5 * (torch.arange(s, device="cuda") // 128))[:, None]
    k, v = (normal(gen, b, h, s, d, dtype=torch.float32) * grow).bfloat16(), normal(gen, b, h, s, d, dtype=torch.bfloat16)
    for softcap in (None, 5.0):
        seen = ref.visible(b, s, s, causal=True, device="cuda")
        want = ref.attention(q, k, v, scale=scale, softcap=softcap, seen=seen, grad_out=do)
        out, lse = ops.score_attention(q, k, v, scale=scale, softcap=softcap, causal_mask=True, return_lse=True)
        within(out, want["out"], want["out_tol"], ("out", scale, softcap))
        within(lse, want["lse"], want["lse_tol"], ("lse", scale, softcap))
        for name, g in zip(("dq", "dk", "dv"), ops.score_attention_grad(do, q, k, v, out, lse, scale=scale, softcap=softcap, causal_mask=True)):
            within(g, want[name], want[name + "_tol"], (name, scale, softcap))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf")])
def test_anything_may_lie_outside_the_documents(ops, d, garbage):
    """A padded batch whose padding rows hold NaN or infinities, in the operands and in the result's gradient."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    b, h, hk, s = 3, 4, 2, 330
    q, do = (normal(gen, b, h, s, d, dtype=torch.bfloat16) for _ in range(2))
    k, v = (normal(gen, b, hk, s, d, dtype=torch.bfloat16) for _ in range(2))
    offs = offsets([[0, 100, 200], [17, 129, 301], [0, 0, 0]])
    for e in range(b):
        for t in (q, do, k, v):
            t[e, :, : int(offs[e, 0])] = garbage
            t[e, :, int(offs[e, -1]):] = garbage
    for causal in (False, True):
        seen = ref.visible(b, s, s, causal=causal, document_offsets=offs, device="cuda")
        want = ref.attention(q, k, v, seen=seen, grad_out=do)
        out, lse = ops.score_attention(q, k, v, causal_mask=causal, document_offsets=offs, return_lse=True)
        within(out, want["out"], want["out_tol"], ("out", d, causal))
        within(lse, want["lse"], want["lse_tol"], ("lse", d, causal))
        for name, g in zip(("dq", "dk", "dv"), ops.score_attention_grad(do, q, k, v, out, lse, causal_mask=causal, document_offsets=offs)):
            within(g, want[name], want[name + "_tol"], (name, d, causal))


def test_odd_strides_offsets_and_out(ops):
    """Views that TMA cannot describe are copied or take the plain kernel; `out` may be a strided or unaligned view, whose
    neighbours stay as they were."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    b, h, s, d = 2, 2, 150, 64
    plain = [normal(gen, b, h, s, d, dtype=torch.bfloat16) for _ in range(3)]
    want = ops.score_attention(*plain, causal_mask=True)
    wide = [torch.zeros(b, h, s, d + 3, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    for w, t in zip(wide, plain):
        w[..., 1:d + 1] = t
    assert torch.equal(ops.score_attention(*[w[..., 1:d + 1] for w in wide], causal_mask=True), want)
    spread = [torch.zeros(b, h, s, 2 * d, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    for w, t in zip(spread, plain):
        w[..., ::2] = t
    assert torch.equal(ops.score_attention(*[w[..., ::2] for w in spread], causal_mask=True), want)
    frame = torch.full((b, s + 2, h, d + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    into = frame[:, 1:s + 1, :, 8:d + 8].transpose(1, 2)
    assert ops.score_attention(*plain, causal_mask=True, out=into).data_ptr() == into.data_ptr()
    assert torch.equal(into, want)
    into.fill_(7.0)
    assert (frame == 7.0).all()
    odd = torch.full((b, h, s, d + 1), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.score_attention(*plain, causal_mask=True, out=odd[..., 1:])
    assert (odd[..., 0] == 7.0).all() and (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    # one key head shown to every batch entry and head by expand()
    k1, v1 = (normal(gen, 1, 1, s, d, dtype=torch.bfloat16) for _ in range(2))
    got = ops.score_attention(plain[0], k1.expand(b, h, s, d), v1.expand(b, h, s, d), causal_mask=True)
    assert torch.equal(got, ops.score_attention(plain[0], k1.expand(b, h, s, d).contiguous(), v1.expand(b, h, s, d).contiguous(), causal_mask=True))


def test_empty_extents(ops):
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    assert ops.score_attention(z(0, 2, 5, 64), z(0, 2, 5, 64), z(0, 2, 5, 64)).shape == (0, 2, 5, 64)
    assert ops.score_attention(z(2, 2, 0, 64), z(2, 2, 5, 64), z(2, 2, 5, 64)).shape == (2, 2, 0, 64)
    out, lse = ops.score_attention(z(2, 2, 5, 64) + 1, z(2, 1, 0, 64), z(2, 1, 0, 64), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv = ops.score_attention_grad(z(2, 2, 5, 64) + 1, z(2, 2, 5, 64), z(2, 1, 0, 64), z(2, 1, 0, 64), out, lse)
    assert (dq == 0).all() and dk.shape == dv.shape == (2, 1, 0, 64)
    empty = z(2, 2, 0, 64)
    dq, dk, dv = ops.score_attention_grad(empty, empty, z(2, 1, 5, 64) + 1, z(2, 1, 5, 64) + 1, empty, torch.zeros(2, 2, 0, device="cuda"))
    assert dq.shape == (2, 2, 0, 64) and (dk == 0).all() and (dv == 0).all()
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    assert ops.score_attention_decode(z(0, 2, 64), z(0, 2, 5, 64), z(0, 2, 5, 64), i32(0)).shape == (0, 2, 64)
    assert (ops.score_attention_decode(z(3, 2, 64) + 1, z(3, 2, 0, 64), z(3, 2, 0, 64), i32(3)) == 0).all()


def test_autograd_form(ops):
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, do = normal(gen, 2, 4, 150, 64, dtype=torch.float16), normal(gen, 2, 4, 150, 64, dtype=torch.float16)
    k, v = (normal(gen, 2, 2, 150, 64, dtype=torch.float16) for _ in range(2))
    opt = dict(causal_mask=True, softcap=10.0, alibi_slopes=torch.tensor([0.5, 0.25, 0.125, 0.1], device="cuda"))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ops.score_attention_trainable(*leaves, **opt)
    got = torch.autograd.grad(out, leaves, do)
    plain, lse = ops.score_attention(q, k, v, return_lse=True, **opt)
    assert torch.equal(out, plain)
    for g, w in zip(got, ops.score_attention_grad(do, q, k, v, plain, lse, **opt)):
        assert torch.equal(g, w)
    # one key head broadcast over batch and heads: autograd sums its gradient
    one = normal(gen, 1, 1, 150, 64, dtype=torch.float16).requires_grad_()
    out = ops.score_attention_trainable(q, one.expand(2, 4, 150, 64), v.repeat_interleave(2, 1), **opt)
    (g1,) = torch.autograd.grad(out, [one], do)
    _, lse = ops.score_attention(q, one.detach().expand(2, 4, 150, 64), v.repeat_interleave(2, 1), return_lse=True, **opt)
    full = ops.score_attention_grad(do, q, one.detach().expand(2, 4, 150, 64), v.repeat_interleave(2, 1), out.detach(), lse, **opt)[1]
    want = full.double().sum((0, 1), keepdim=True)
    # autograd adds the eight gradients in fp16: each of the sums' seven roundings is at most half a step of a partial sum
    assert ((g1.double() - want).abs() <= 8 * 2.0 ** -11 * full.double().abs().sum((0, 1), keepdim=True) + 2.0 ** -20).all()
    # differences along one direction, through the operator in float32
    leaves = [t.float().requires_grad_() for t in (q, k, v)]
    out = ops.score_attention_trainable(*leaves, **opt)
    grads = torch.autograd.grad((out * do.float()).sum(), leaves)
    for which in range(3):
        step = torch.randn(leaves[which].shape, generator=gen, device="cuda") * 1e-2
        ends = []
        for sign in (1.0, -1.0):
            moved = [t.detach() for t in leaves]
            moved[which] = moved[which] + sign * step
            ends.append((ops.score_attention(*moved, **opt).double() * do.double()).sum())
        want, got = float((ends[0] - ends[1]) / 2), float((grads[which].double() * step.double()).sum())
        # the third-order term of a step of 1e-2 and fp32 rounding of some 1e5 terms stay below 1e-3 of the terms' norm
        assert abs(want - got) <= 1e-3 * float(grads[which].double().norm() * step.double().norm()), which


def test_first_call_of_a_host_thread(ops):
    """A host thread whose first CUDA call is one of these operators (an autograd backward thread, a server's worker)."""
    import threading
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, do = (normal(gen, 1, 2, 100, 64, dtype=torch.float16) for _ in range(2))
    out, lse = ops.score_attention(q, q, q, return_lse=True)
    want = ops.score_attention_grad(do, q, q, q, out, lse)
    a, b = normal(gen, 64, 64, dtype=torch.bfloat16), normal(gen, 64, 64, dtype=torch.bfloat16)
    product = ops.fused_matmul(a, b)
    got = {}

    def work(name, call):
        try:
            got[name] = call()
        except Exception as e:                                        # reported below, in the test's own thread
            got[name] = e

    for name, call in (("grad", lambda: ops.score_attention_grad(do, q, q, q, out, lse)), ("forward", lambda: ops.score_attention(q, q, q)),
                       ("product", lambda: ops.fused_matmul(a, b))):
        t = threading.Thread(target=work, args=(name, call))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got["grad"], want))
    assert torch.equal(got["forward"], out) and torch.equal(got["product"], product)


def test_streams_and_graphs(ops):
    """Calls on two side streams at once, and forward + backward captured into two graphs that replay after new inputs were written."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    sets = [[normal(gen, 1, 4, 300, 64, dtype=torch.bfloat16) for _ in range(4)] for _ in range(2)]
    lengths = torch.tensor([200], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        out, lse = ops.score_attention(q, k, v, causal_mask=True, softcap=20.0, return_lse=True)
        token = ops.score_attention_decode(q[:, :, 0], k, v, lengths)
        shared = ops.shared_prefix_attention(q[:, :, 1], k[0], v[0], k, v, lengths)
        return (out, token, shared, *ops.score_attention_grad(do, q, k, v, out, lse, causal_mask=True, softcap=20.0))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    graphs, held = [], []
    for s in sets:
        static = [t.clone() for t in s]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*static)
        graphs.append(g)
        held.append((static, res))
    for turn in range(3):
        for n, (static, _) in enumerate(held):
            for t, src in zip(static, sets[(n + turn) % 2]):
                t.copy_(src)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):            # both at once: no scratch is shared between them
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for n, (_, res) in enumerate(held):
            assert all(torch.equal(a, b) for a, b in zip(res, want[(n + turn) % 2])), turn


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------
def token_and_check(ops, gen, dtype, b, h, hk, s, d, lengths, prefix=0, softcap=None, alibi=False, layout="bhsd", factor=1.0, scale=None):
    q = normal(gen, b, h, d, dtype=dtype, factor=factor)
    k, v = (normal(gen, b, hk, s, d, dtype=dtype, layout=layout) for _ in range(2))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for e, n in enumerate(lengths):                                  # what lies behind a request's rows is arbitrary
        k[e, :, max(n, 0):] = float("nan")
        v[e, :, max(n, 0):] = float("inf")
    slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if alibi else None
    opt = dict(scale=scale, softcap=softcap)
    pk = pv = None
    if prefix:
        pk, pv = (normal(gen, hk, prefix, d, dtype=dtype) for _ in range(2))
        out, lse = ops.shared_prefix_attention(q, pk, pv, k, v, lens, alibi_slopes=slopes, return_lse=True, **opt)
    else:
        out, lse = ops.score_attention_decode(q, k, v, lens, alibi_slopes=slopes, return_lse=True, **opt)
    want = ref.token_attention(q, k, v, lengths, prefix_k=pk, prefix_v=pv, slopes=slopes, **opt)
    what = (str(dtype), b, h, hk, s, d, prefix, softcap, alibi, layout)
    within(out, want["out"], want["out_tol"], ("out", *what))
    within(lse, want["lse"], want["lse_tol"], ("lse", *what))


TOKENS = [
    # b, h, hk, cache rows, d, lengths, softcap, alibi, layout
    (1, 1, 1, 1, 64, [1], None, False, "bhsd"),
    (3, 2, 1, 17, 128, [0, 1, 17], None, True, "bhsd"),
    (2, 8, 2, 700, 128, [700, 333], 20.0, True, "bshd"),
    (4, 7, 1, 300, 64, [1, 63, 64, 65], None, True, "bhsd"),
    (2, 16, 1, 1000, 128, [1000, 129], None, False, "bshd"),
    (1, 32, 8, 5000, 128, [4999], None, True, "bhsd"),
    (2, 3, 3, 2000, 96, [2000, 40], 15.0, False, "bhsd"),
    (2, 40, 2, 260, 80, [260, 128], None, False, "bshd"),
    (1, 2, 2, 40000, 64, [39990], None, False, "bhsd"),
    (3, 4, 4, 200, 64, [-5, 100, 900], 30.0, False, "bhsd"),          # lengths outside the cache are clamped
    (5, 130, 1, 150, 64, [150, 3, 0, 77, 149], None, False, "bhsd"),
    (2, 4, 2, 90, 33, [90, 50], 10.0, True, "bhsd"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", TOKENS, ids=lambda c: "-".join(map(str, c)))
def test_tokens(ops, dtype, case):
    b, h, hk, s, d, lengths, softcap, alibi, layout = case
    gen = torch.Generator(device="cuda").manual_seed(20 + s)
    token_and_check(ops, gen, DT[dtype], b, h, hk, s, d, lengths, 0, softcap, alibi, layout, factor=3.0 if softcap else 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("prefix", [1, 64, 130, 1500])
@pytest.mark.parametrize("case", [TOKENS[i] for i in (0, 1, 2, 3, 4, 7, 9, 10, 11)], ids=lambda c: "-".join(map(str, c)))
def test_tokens_behind_a_shared_prefix(ops, dtype, prefix, case):
    b, h, hk, s, d, lengths, softcap, alibi, layout = case
    gen = torch.Generator(device="cuda").manual_seed(30 + s + prefix)
    token_and_check(ops, gen, DT[dtype], b, h, hk, s, d, lengths, prefix, softcap, alibi, layout, factor=3.0 if softcap else 1.0)


STREAMED = [
    # b, h, hk, cache rows, d, lengths: more 64-key units than blocks, in every kind of raggedness
    (3, 32, 8, 4100, 128, lambda e: [4100, 0, 1][e % 3]),
    (70, 8, 4, 900, 64, lambda e: (e * 37) % 901),
    (40, 40, 2, 1300, 128, lambda e: 1300 if e == 39 else 0),          # all work in the last entry, two row tiles
    (9, 4, 4, 5000, 96, lambda e: [64, 63, 65, 128, 5000, 4999, 0, 2, 777][e]),
    (33, 16, 16, 800, 64, lambda e: 1),                                # fewer units than blocks
    (34, 8, 8, 1000, 128, lambda e: 0),                                # no work at all
]


@pytest.mark.parametrize("prefix", [0, 70, 6000])
@pytest.mark.parametrize("case", STREAMED, ids=lambda c: "-".join(map(str, c[:5])))
def test_streamed_caches(ops, case, prefix):
    b, h, hk, s, d, length = case
    gen = torch.Generator(device="cuda").manual_seed(50 + s)
    token_and_check(ops, gen, torch.bfloat16, b, h, hk, s, d, [length(e) for e in range(b)], prefix, None, prefix == 0)


def test_which_kernel_runs(ops, binding):
    """16-bit tensors run on the tensor cores in every form; nothing falls back unseen."""
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16), (80, torch.bfloat16)):
        q, k = torch.randn(1, 4, 130, d, device="cuda").to(dtype), torch.randn(1, 2, 130, d, device="cuda").to(dtype)
        size = "d128" if d > 64 else "d64"
        out, lse = ops.score_attention(q, k, k, causal_mask=True, softcap=30.0, return_lse=True)
        assert binding.last_kernel_name() == f"score_attention_tcgen05_{size}"
        ops.score_attention_grad(out, q, k, k, out, lse, causal_mask=True, softcap=30.0)
        assert binding.last_kernel_name() == f"score_attention_grad_tcgen05_{size}"
        n = torch.tensor([130], dtype=torch.int32, device="cuda")
        ops.score_attention_decode(q[:, :, 0], k, k, n)
        assert binding.last_kernel_name() == f"score_attention_decode_{size}"
        before = binding.launch_count()
        big = torch.randn(64, 8, d, device="cuda").to(dtype)
        cache = torch.randn(64, 2, 20, d, device="cuda").to(dtype)
        common = torch.randn(2, 40000, d, device="cuda").to(dtype)
        ops.shared_prefix_attention(big, common, common, cache, cache, torch.full((64,), 20, dtype=torch.int32, device="cuda"))
        assert binding.launch_count() == before + 3                    # prefix on the tcgen05 kernel, caches, join
    ops.score_attention(q.float(), k.float(), k.float())
    assert binding.last_kernel_name() == "score_attention_simt"


def test_split_gradient_streams(ops):
    """Few key tiles that many query heads share: the key blocks' streams are cut into parts, of one head or of several."""
    gen = torch.Generator(device="cuda").manual_seed(60)
    for b, h, hk, s, d, kind in ((1, 16, 1, 700, 128, "causal"), (1, 2, 2, 3000, 64, "causal"), (2, 6, 1, 900, 96, "documents_causal"),
                                 (1, 8, 2, 1100, 128, "prefix")):
        train_and_check(ops, gen, torch.bfloat16, b, h, hk, s, s, d, kind, None, d == 64)


@pytest.mark.parametrize("prefix", [300, 5000])
def test_large_batches_behind_a_shared_prefix(ops, prefix):
    gen = torch.Generator(device="cuda").manual_seed(40)
    for b, h, hk, d, dtype in ((64, 8, 2, 128, torch.bfloat16), (100, 6, 2, 64, torch.float16), (37, 14, 2, 128, torch.bfloat16)):
        token_and_check(ops, gen, dtype, b, h, hk, 70, d, [(13 * e) % 71 for e in range(b)], prefix, 20.0 if d == 64 else None, True)


def test_prefix_and_caches_overlap_in_order(ops):
    """The caches' launch may begin while the prefix's still runs: results stay those of the ordered calls, back to back on changing
    inputs, on two streams and in a replayed graph, and what is queued behind sees them complete."""
    gen = torch.Generator(device="cuda").manual_seed(45)
    b, h, hk, d, p, s = 64, 16, 4, 128, 9000, 900
    sets = []
    for _ in range(3):
        q = normal(gen, b, h, d, dtype=torch.bfloat16)
        pk, pv = (normal(gen, hk, p, d, dtype=torch.bfloat16) for _ in range(2))
        k, v = (normal(gen, b, hk, s, d, dtype=torch.bfloat16) for _ in range(2))
        sets.append((q, pk, pv, k, v, torch.randint(0, s + 1, (b,), generator=gen, device="cuda").int()))
    sets[2][5].zero_()                                                 # no request has keys of its own: the caches' blocks end at once
    want = []
    for args in sets:
        torch.cuda.synchronize()
        want.append(ops.shared_prefix_attention(*args).clone())
        torch.cuda.synchronize()
    ref_out = ref.token_attention(*[sets[0][i] for i in (0, 3, 4)], sets[0][5].tolist(), prefix_k=sets[0][1], prefix_v=sets[0][2])
    within(want[0], ref_out["out"], ref_out["out_tol"], "overlap")
    for _ in range(10):
        got = [ops.shared_prefix_attention(*args).float() * 2 for args in sets for _ in range(2)]
        assert all(torch.equal(g, want[i // 2].float() * 2) for i, g in enumerate(got))
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.shared_prefix_attention(*static).float() * 2
    for turn in range(6):
        for t, src in zip(static, sets[turn % 3]):
            t.copy_(src)
        graph.replay()
        assert torch.equal(res, want[turn % 3].float() * 2), turn
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.shared_prefix_attention(*sets[i % 3]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(outs))


def test_prefix_form_equals_the_cache_form(ops):
    """The same keys as one cache and as prefix + cache give the same result up to the join's rounding; no prefix is the cache form itself."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    b, h, hk, d, p, s = 5, 8, 2, 128, 700, 90
    q = normal(gen, b, h, d, dtype=torch.bfloat16)
    pk, pv = (normal(gen, hk, p, d, dtype=torch.bfloat16) for _ in range(2))
    k, v = (normal(gen, b, hk, s, d, dtype=torch.bfloat16) for _ in range(2))
    lens = torch.tensor([90, 0, 1, 44, 89], dtype=torch.int32, device="cuda")
    got = ops.shared_prefix_attention(q, pk, pv, k, v, lens).double()
    joined = [torch.cat([a[None].expand(b, hk, p, d), c], 2) for a, c in ((pk, k), (pv, v))]
    whole = ops.score_attention_decode(q, *joined, lens + p).double()
    # both round P and the result to bf16: (u + u) of the weighted mass, which |v| <= 6 bounds by 6 in all
    assert ((got - whole).abs() <= 4 * 2.0 ** -8 * 6).all() and (got - whole).norm() <= 2 * 2.0 ** -8 * whole.norm()
    none = torch.empty(hk, 0, d, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(ops.shared_prefix_attention(q, none, none, k, v, lens), ops.score_attention_decode(q, k, v, lens))


def test_decode_follows_the_prompt_form(ops):
    """A prompt, then its tokens one by one through a growing cache: the used-together path.  Both forms agree within their bounds."""
    gen = torch.Generator(device="cuda").manual_seed(42)
    h, hk, d, n, more = 8, 2, 128, 100, 6
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(h)], device="cuda")
    q = normal(gen, 1, h, n + more, d, dtype=torch.bfloat16, factor=2.0)
    k, v = (normal(gen, 1, hk, n + more, d, dtype=torch.bfloat16) for _ in range(2))
    seen = ref.visible(1, n + more, n + more, causal=True, device="cuda")
    want = ref.attention(q, k, v, softcap=25.0, slopes=slopes, seen=seen)
    prompt = ops.score_attention(q[:, :, :n], k[:, :, :n], v[:, :, :n], causal_mask=True, softcap=25.0, alibi_slopes=slopes)
    within(prompt, want["out"][:, :, :n], want["out_tol"][:, :, :n], "prompt")
    cache = [torch.full((1, hk, 256, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for c, t in zip(cache, (k, v)):
        c[:, :, :n] = t[:, :, :n]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for t in range(n, n + more):
        for c, src in zip(cache, (k, v)):
            c[:, :, t] = src[:, :, t]
        lens += 1
        token = ops.score_attention_decode(q[:, :, t], *cache, lens, softcap=25.0, alibi_slopes=slopes)
        within(token, want["out"][:, :, t], want["out_tol"][:, :, t], t)
        shared = ops.shared_prefix_attention(q[:, :, t], k[0, :, :n], v[0, :, :n], cache[0][:, :, n:], cache[1][:, :, n:], lens - n, softcap=25.0,
                                             alibi_slopes=slopes)
        within(shared, want["out"][:, :, t], want["out_tol"][:, :, t], ("shared", t))


def test_offsets_beyond_32_bits(ops):
    """A cache and a prompt whose last entry begins more than 2^31 elements behind the first."""
    gen = torch.Generator(device="cuda").manual_seed(43)
    hk, s, d = 2, 300, 64
    far = (1 << 31) + (1 << 20)
    flat = torch.empty(far + hk * s * d, dtype=torch.bfloat16, device="cuda")
    for shape_kv in ("cache",):
        kv = flat.as_strided((2, hk, s, d), (far, s * d, d, 1))
        kv.copy_(normal(gen, 2, hk, s, d, dtype=torch.bfloat16))
        near = kv.contiguous()
        q = normal(gen, 2, 4, d, dtype=torch.bfloat16)
        lens = torch.tensor([300, 211], dtype=torch.int32, device="cuda")
        assert torch.equal(ops.score_attention_decode(q, kv, kv, lens), ops.score_attention_decode(q, near, near, lens))
        qs = normal(gen, 2, 4, s, d, dtype=torch.bfloat16)
        out, lse = ops.score_attention(qs, kv, kv, causal_mask=True, return_lse=True)
        want, lse_w = ops.score_attention(qs, near, near, causal_mask=True, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, lse_w)
        assert all(torch.equal(a, b) for a, b in zip(ops.score_attention_grad(qs, qs, kv, kv, out, lse, causal_mask=True),
                                                     ops.score_attention_grad(qs, qs, near, near, out, lse, causal_mask=True)))
    # rows more than 2^31 elements apart inside one head
    rows = flat.as_strided((1, 1, 2, d), (0, 0, far, 1))
    rows.copy_(normal(gen, 1, 1, 2, d, dtype=torch.bfloat16))
    q, two = normal(gen, 1, 1, d, dtype=torch.bfloat16), torch.tensor([2], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.score_attention_decode(q, rows, rows, two), ops.score_attention_decode(q, rows.contiguous(), rows.contiguous(), two))


def test_token_out_and_layouts(ops):
    gen = torch.Generator(device="cuda").manual_seed(44)
    b, h, hk, s, d = 3, 4, 2, 130, 64
    q, (k, v) = normal(gen, b, h, d, dtype=torch.float16), [normal(gen, b, hk, s, d, dtype=torch.float16) for _ in range(2)]
    lens = torch.tensor([130, 5, 64], dtype=torch.int32, device="cuda")
    want = ops.score_attention_decode(q, k, v, lens)
    wide = torch.zeros(b, hk, s + 3, d + 1, dtype=torch.float16, device="cuda")
    wide[:, :, 2:s + 2, 1:] = k
    assert torch.equal(ops.score_attention_decode(q, wide[:, :, 2:s + 2, 1:], v, lens), want)
    frame = torch.full((h, b, d + 8), 3.0, dtype=torch.float16, device="cuda")
    into = frame[..., 8:].transpose(0, 1)
    ops.score_attention_decode(q, k, v, lens, out=into)
    assert torch.equal(into, want) and (frame[..., :8] == 3.0).all()
    if torch.cuda.device_count() > 1:
        with torch.cuda.device(0):
            there = [t.to("cuda:1") for t in (q, k, v, lens)]
            assert torch.equal(ops.score_attention_decode(*there).to("cuda:0"), want)
