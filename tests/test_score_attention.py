"""CPU tests of the score-modified attention: the 64-bit reference against differences and autograd, the descriptor's
layout, and what the Python surface and the C entry points refuse before they touch a device."""
import ctypes
import inspect

import pytest
import torch

from oracle import score_attention as ref


def _inputs(b=2, h=4, hk=2, sq=5, sk=7, d=8, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)
                 for shape in ((b, h, sq, d), (b, hk, sk, d), (b, hk, sk, d), (b, h, sq, d)))


@pytest.mark.parametrize("softcap", [None, 1.5])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix", "documents", "documents_causal"])
def test_reference_gradients_match_autograd_and_differences(mask, softcap):
    q, k, v, do = _inputs()
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0], dtype=torch.float64)
    seen = ref.visible(2, 5, 7, causal=mask in ("causal", "prefix", "documents_causal"),
                       prefix_lengths=torch.tensor([3, 7]) if mask == "prefix" else None,
                       document_offsets=torch.tensor([[0, 3, 3, 6], [1, 4, 7, 7]]) if "documents" in mask else None)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    got = ref.attention(q, k, v, softcap=softcap, slopes=slopes, seen=seen, grad_out=do)

    def scalar(a, b_, c):
        return (ref.attention(a, b_, c, softcap=softcap, slopes=slopes, seen=seen)["out"] * do).sum()

    # rows without keys are NaN in autograd's logsumexp gradient: compare through torch only where every row sees a key
    if mask in ("full", "causal", "prefix"):
        want = torch.autograd.grad(scalar(*leaves), leaves)
        for name, w in zip(("dq", "dk", "dv"), want):
            assert torch.allclose(got[name], w, rtol=1e-10, atol=1e-12), name
    # central differences in 64 bits: h = 1e-5 leaves h^2 ~ 1e-10 of the third derivative and 1e-16 / h ~ 1e-11 of rounding
    step = 1e-5
    rng = torch.Generator().manual_seed(5)
    for which, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn(leaves[which].shape, generator=rng, dtype=torch.float64)
        ends = []
        for sign in (1.0, -1.0):
            moved = [q, k, v]
            moved[which] = moved[which] + sign * step * direction
            ends.append(scalar(*moved))
        slope = (ends[0] - ends[1]) / (2 * step)
        assert abs(float(slope - (got[name] * direction).sum())) < 1e-7, name


def test_reference_rows_without_keys_are_zero():
    q, k, v, do = _inputs(sq=7, sk=4)                      # causal with more queries than keys: three rows see nothing
    seen = ref.visible(2, 7, 4, causal=True)
    got = ref.attention(q, k, v, seen=seen, grad_out=do)
    assert (got["out"][:, :, :3] == 0).all() and (got["lse"][:, :, :3] == -float("inf")).all() and (got["dq"][:, :, :3] == 0).all()
    assert all(torch.isfinite(got[n]).all() for n in ("out", "dq", "dk", "dv"))


def test_signatures(ops):
    for name in ("score_attention", "score_attention_grad", "score_attention_trainable", "score_attention_decode", "shared_prefix_attention"):
        assert name in ops.__all__
    options = ["scale", "causal_mask", "softcap", "alibi_slopes", "document_offsets", "prefix_lengths"]
    assert list(inspect.signature(ops.score_attention).parameters) == ["query", "key", "value", *options, "return_lse", "out"]
    assert list(inspect.signature(ops.score_attention_grad).parameters) == ["grad_out", "query", "key", "value", "out", "lse", *options]
    assert list(inspect.signature(ops.score_attention_trainable).parameters) == ["query", "key", "value", *options]


def _bad_sequences():
    q, k, v, _ = _inputs(dtype=torch.float32)
    i32 = dict(dtype=torch.int32)
    return {
        "rank": ((q[0], k, v), {}, ValueError),
        "dtype": ((q.double(), k.double(), v.double()), {}, ValueError),
        "mixed dtype": ((q, k.half(), v), {}, ValueError),
        "not a tensor": ((q, k.numpy(), v), {}, TypeError),
        "head groups": ((q[:, :3], k, v), {}, ValueError),
        "head dim": ((q, k[..., :4], v), {}, ValueError),
        "key length": ((q, k, v[:, :, :3]), {}, ValueError),
        "wide heads": (tuple(torch.zeros(1, 1, 2, 257) for _ in range(3)), {}, ValueError),
        "softcap 0": ((q, k, v), dict(softcap=0.0), ValueError),
        "softcap < 0": ((q, k, v), dict(softcap=-3.0), ValueError),
        "softcap nan": ((q, k, v), dict(softcap=float("nan")), ValueError),
        "scale nan": ((q, k, v), dict(scale=float("nan")), ValueError),
        "slopes shape": ((q, k, v), dict(alibi_slopes=torch.zeros(2)), ValueError),
        "slopes dtype": ((q, k, v), dict(alibi_slopes=torch.zeros(4).half()), ValueError),
        "offsets dtype": ((q, k, v), dict(document_offsets=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
        "offsets batch": ((q, k, v), dict(document_offsets=torch.zeros(1, 3, **i32)), ValueError),
        "offsets rank": ((q, k, v), dict(document_offsets=torch.zeros(3, **i32)), ValueError),
        "offsets single": ((q, k, v), dict(document_offsets=torch.zeros(2, 1, **i32)), ValueError),
        "offsets strided": ((q, k, v), dict(document_offsets=torch.zeros(2, 6, **i32)[:, ::2]), ValueError),
        "prefix alone": ((q, k, v), dict(prefix_lengths=torch.zeros(2, **i32)), ValueError),
        "prefix shape": ((q, k, v), dict(prefix_lengths=torch.zeros(3, **i32), causal_mask=True), ValueError),
        "prefix and documents": ((q, k, v), dict(prefix_lengths=torch.zeros(2, **i32), causal_mask=True,
                                                 document_offsets=torch.zeros(2, 3, **i32)), ValueError),
    }


@pytest.mark.parametrize("name", sorted(_bad_sequences()))
def test_sequence_forms_refuse(ops, name):
    args, options, error = _bad_sequences()[name]
    with pytest.raises(error):
        ops.score_attention(*args, **options)
    with pytest.raises(error):
        ops.score_attention_trainable(*args, **options)
    if name not in ("rank", "not a tensor"):
        with pytest.raises(error):
            ops.score_attention_grad(args[0], *args, args[0], torch.zeros(args[0].shape[:3]), **options)


def test_token_forms_refuse(ops):
    q, k, v = torch.zeros(2, 4, 8), torch.zeros(2, 2, 6, 8), torch.zeros(2, 2, 6, 8)
    lengths, pk = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, 8)
    bad = [
        ((q[0], k, v, lengths), {}), ((q, k[0], v, lengths), {}), ((q[:, :3], k, v, lengths), {}), ((q, k, v[:, :, :5], lengths), {}),
        ((q, k, v, lengths.long()), {}), ((q, k, v, lengths[:1]), {}), ((q.double(), k.double(), v.double(), lengths), {}),
        ((q, k, v, lengths), dict(softcap=0.0)), ((q, k, v, lengths), dict(alibi_slopes=torch.zeros(3))),
    ]
    for args, options in bad:
        with pytest.raises(ValueError):
            ops.score_attention_decode(*args, **options)
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(args[0], pk.to(args[0].dtype), pk.to(args[0].dtype), *args[1:], **options)
    for prefix in ((pk[:1], pk[:1]), (pk, pk[:, :2]), (pk[..., :4], pk[..., :4]), (pk.half(), pk.half()), (pk[0], pk[0])):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(q, *prefix, k, v, lengths)
    with pytest.raises(TypeError):
        ops.score_attention_decode(q, k, v, [1, 2])


def test_packed_descriptor_has_the_structs_layout(binding):
    """The one-call packing writes every field where the struct has it."""
    pack, fields = binding.SCORE_ATTENTION_PACK, binding.SM120ScoreAttentionDesc._fields_
    assert pack.size == ctypes.sizeof(binding.SM120ScoreAttentionDesc)
    values, expect = [], []
    for name, kind in fields:
        count = getattr(kind, "_length_", 1)
        own = [float(len(values) + i) if kind is ctypes.c_float else len(values) + i + 1 for i in range(count)]
        values += own
        expect.append((name, own if count > 1 else own[0]))
    d = binding.SM120ScoreAttentionDesc.from_buffer(bytearray(pack.pack(*values)))
    for name, want in expect:
        got = getattr(d, name)
        assert (list(got) if isinstance(want, list) else got) == want, name


def test_packed_descriptor_reaches_the_entry_points(binding):
    d = _good(binding, "grad")
    d.workspace, d.workspace_bytes = None, 0
    packed = bytes(d)
    assert packed[-binding.SCORE_ATTENTION_TAIL.size:] == binding.SCORE_ATTENTION_TAIL.pack(0, 0, 0)
    assert binding.score_attention_call(LAUNCH["grad"])(packed) == 1              # no workspace
    assert binding.score_attention_call(LAUNCH["forward"])(b"\0" * len(packed)) == 1


def test_needs_a_gpu(ops):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    q, k, v, _ = _inputs(dtype=torch.float32)
    with pytest.raises(ops.UnimplementedError):
        ops.score_attention(q, k, v)
    with pytest.raises(ops.UnimplementedError):
        ops.score_attention_decode(q[:, :, 0], k, v, torch.ones(2, dtype=torch.int32))


def _good(binding, form):
    d = binding.new_score_attention_desc()
    d.batch, d.heads, d.kv_heads, d.seq_q, d.seq_k, d.head_dim = 2, 4, 2, 1 if form == "decode" else 16, 32, 64
    d.dtype = binding.DTYPE_BFLOAT16
    d.q, d.k, d.v, d.out, d.lse = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000      # never dereferenced: every case is rejected first
    if form == "grad":
        d.grad_out, d.grad_q, d.grad_k, d.grad_v = 0x6000, 0x7000, 0x8000, 0x9000
        d.workspace, d.workspace_bytes = 0x10000, 1 << 40
    if form == "decode":
        d.key_lengths = 0xA000
        d.workspace, d.workspace_bytes = 0x10000, 1 << 40
    return d


LAUNCH = {"forward": "sm120_launch_score_attention", "grad": "sm120_launch_score_attention_grad", "decode": "sm120_launch_score_attention_decode"}


@pytest.mark.parametrize("form", sorted(LAUNCH))
@pytest.mark.parametrize("field, value", [
    ("struct_size", 8), ("dtype", 3), ("dtype", -1), ("batch", -1), ("batch", 65536), ("heads", 0), ("heads", 3), ("kv_heads", 0),
    ("seq_k", -1), ("seq_k", 1 << 30), ("head_dim", 0), ("head_dim", 257), ("softcap", -1.0), ("softcap", float("nan")),
    ("scale", float("nan")), ("num_documents", -1), ("num_documents", 3), ("prefix_lengths", 0xB000), ("q", None), ("k", None), ("out", None),
    ("q_stride", (-1, 0, 0)), ("prefix_len", -1),
])
def test_c_entry_points_refuse_without_a_device(binding, form, field, value):
    lib, d = binding.load_library(), _good(binding, form)
    if isinstance(value, tuple):
        getattr(d, field)[:] = value
    else:
        setattr(d, field, value)
    assert getattr(lib, LAUNCH[form])(ctypes.byref(d)) == 1
    assert lib.sm120_score_attention_grad_workspace_bytes(ctypes.byref(d)) == 0 or form != "grad"


def test_c_entry_points_refuse_what_belongs_to_another_form(binding):
    lib = binding.load_library()
    for form, field, value in (("forward", "key_lengths", 0xA000), ("forward", "prefix_len", 4), ("grad", "lse", None), ("grad", "grad_out", None),
                               ("grad", "grad_k", None), ("grad", "workspace", None), ("grad", "workspace", 0x10008), ("grad", "workspace_bytes", 64),
                               ("decode", "seq_q", 2), ("decode", "causal", 1), ("decode", "key_lengths", None), ("decode", "prefix_len", 4)):
        d = _good(binding, form)
        setattr(d, field, value)
        assert getattr(lib, LAUNCH[form])(ctypes.byref(d)) == 1, (form, field)
    for form, field in (("forward", "out_stride"), ("decode", "out_stride"), ("grad", "grad_q_stride"), ("grad", "grad_k_stride"), ("grad", "grad_v_stride")):
        d = _good(binding, form)
        for name in ("out_stride", "grad_q_stride", "grad_k_stride", "grad_v_stride"):
            getattr(d, name)[:] = (65536, 8192, 64)
        getattr(d, field)[1] = 0                                                # heads written over one another
        assert getattr(lib, LAUNCH[form])(ctypes.byref(d)) == 1, (form, field)
    assert lib.sm120_launch_score_attention(None) == 1
    d = _good(binding, "forward")
    d.batch = 0
    assert lib.sm120_launch_score_attention(ctypes.byref(d)) == 0               # nothing to do
    assert d.struct_size == ctypes.sizeof(binding.SM120ScoreAttentionDesc)
