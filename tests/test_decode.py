"""CPU tests of the decode-step caller (qorvix_amd/decode.py): the token's GEMV list mirrors the
reference's decoder call order and type mix, its byte accounting is the GGUF arithmetic, and the
plan entry points reject bad handles before touching a device."""
from __future__ import annotations

import qorvix_amd as qvx
from qorvix_amd import decode


def test_layer_call_order_mirrors_reference_decoder():
    # runtime/src/text_model.cpp:146-173: wq, wk, wv, (attention), wo, ffn_gate, ffn_up, ffn_down
    assert [s[0] for s in decode.LAYER_SPECS] == ["wq", "wk", "wv", "wo", "ffn_gate", "ffn_up", "ffn_down"]
    specs = decode.sweep_specs()
    assert len(specs) == 32 * 7 + 1 and specs[-1][1] == "lm_head"
    assert [s[1] for s in specs[:7]] == [s[0] for s in decode.LAYER_SPECS]
    # inputs: q/k/v/gate/up read the normed state, wo the attention output, ffn_down the SwiGLU output
    assert {s[0]: s[4] for s in decode.LAYER_SPECS} == {
        "wq": "xn", "wk": "xn", "wv": "xn", "wo": "attn", "ffn_gate": "xn", "ffn_up": "xn", "ffn_down": "act"}


def test_q4_k_m_type_mix():
    types = {s[0]: s[3] for s in decode.LAYER_SPECS}
    assert types["wv"] == qvx.Q6_K and types["ffn_down"] == qvx.Q6_K and decode.LM_HEAD[3] == qvx.Q6_K
    assert all(types[n] == qvx.Q4_K for n in ("wq", "wk", "wo", "ffn_gate", "ffn_up"))


def test_sweep_byte_accounting():
    # per-tensor bytes from the block formats: rows * (cols / 256) * {144 (Q4_K), 210 (Q6_K)}
    per = {"wq": 4096 * 16 * 144, "wk": 1024 * 16 * 144, "wv": 1024 * 16 * 210, "wo": 4096 * 16 * 144,
           "ffn_gate": 14336 * 16 * 144, "ffn_up": 14336 * 16 * 144, "ffn_down": 4096 * 56 * 210}
    assert per == {"wq": 9437184, "wk": 2359296, "wv": 3440640, "wo": 9437184, "ffn_gate": 33030144,
                   "ffn_up": 33030144, "ffn_down": 48168960}
    layer = sum(per.values())
    assert layer == 138903552
    lm = 128256 * 16 * 210
    wb, ab1 = decode.sweep_bytes(1)
    _, ab8 = decode.sweep_bytes(8)
    assert wb == 32 * layer + lm == 4875853824
    # activations in + outputs out, 4 bytes each, per GEMV and vector
    io = sum(rows + cols for _, _, rows, cols, _, _ in decode.sweep_specs()) * 4
    assert ab1 == wb + io == 4886868992
    assert ab8 == wb + 8 * io == 4963975168


def test_plan_entry_points_reject_null_handles():
    lib = qvx.lib()
    assert lib.qvx_plan_size(None) == 0
    assert lib.qvx_plan_launch(None, None) == qvx.E_NULL
    assert lib.qvx_plan_run_eager(None, None) == qvx.E_NULL
    assert lib.qvx_plan_instantiate(None) == qvx.E_NULL
    assert lib.qvx_plan_add_qmatmul_n(None, None, None, qvx.Q4_K, None, 1, 16, 256) == qvx.E_NULL
    assert lib.qvx_plan_create(None) == qvx.E_NULL
    lib.qvx_plan_destroy(None)
    assert qvx.strerror(qvx.E_STATE).startswith("plan not instantiated")


def test_fused_model_stacks_same_input_pairs():
    """Model.fused stacks q with k and gate with up (same type and row length) row-wise; calls()
    then yields 5 GEMVs per layer in the reference's order, each stacked weight in place of its
    first part, and the bytes of each part sit where its rows do."""
    import torch
    from qorvix_amd import decode
    m = decode.Model()
    for l in range(2):
        layer = {}
        for i, (name, rows, cols, t, _) in enumerate(decode.LAYER_SPECS):
            rows, cols = rows // 256, cols // 16  # small stand-ins keeping the type mix and ratios
            nb = qvx.weight_bytes(t, rows, cols)
            layer[name] = decode.DevWeight(torch.full((nb,), 16 * l + i, dtype=torch.uint8), t, rows, cols)
        m.layers.append(layer)
    m.lm_head = decode.DevWeight(torch.zeros(qvx.weight_bytes(qvx.Q6_K, 8, 256), dtype=torch.uint8), qvx.Q6_K, 8, 256)
    f = m.fused()
    names = [(l, n, src) for l, n, _, src in f.calls()]
    per_layer = [("wqk", "xn"), ("wv", "xn"), ("wo", "attn"), ("ffn_gateup", "xn"), ("ffn_down", "act")]
    assert names == [(l, n, s) for l in range(2) for n, s in per_layer] + [(2, "lm_head", "xn")]
    for l in range(2):
        qk, gu = f.layers[l]["wqk"], f.layers[l]["ffn_gateup"]
        q, k = m.layers[l]["wq"], m.layers[l]["wk"]
        assert (qk.rows, qk.cols, qk.type) == (q.rows + k.rows, q.cols, q.type)
        assert torch.equal(qk.data[:q.data.numel()], q.data) and torch.equal(qk.data[q.data.numel():], k.data)
        assert gu.rows == m.layers[l]["ffn_gate"].rows + m.layers[l]["ffn_up"].rows
        assert f.layers[l]["wv"] is m.layers[l]["wv"]  # Q6_K: not stacked with q/k, shared
    assert f.parts["wqk"] == (("wq", 16), ("wk", 4))
    # the unfused model keeps the reference's 7 calls per layer
    assert [n for l, n, _, _ in m.calls() if l == 0] == [s[0] for s in decode.LAYER_SPECS]


def test_fused_step_refuses_a_model_without_norms():
    """Every launch of FusedDecodeStep folds an RMSNorm into its activations; a model whose GGUF file
    lacks a norm tensor is refused up front (before any device work) instead of running un-normed."""
    import pytest

    m = decode.Model(lm_head=None, norms=[{"attn_norm": object(), "ffn_norm": None}], output_norm=None)
    m.layers.append({})
    with pytest.raises(ValueError, match="ffn_norm of layer 0"):
        decode.FusedDecodeStep(m, 1)
    m.norms = []
    with pytest.raises(ValueError, match="attn_norm of layer 0"):
        decode.FusedDecodeStep(m, 1)
    m.norms = [{"attn_norm": object(), "ffn_norm": object()}]
    m.lm_head = object()
    with pytest.raises(ValueError, match="output_norm"):
        decode.FusedDecodeStep(m, 1)


def _paged_model(layers=2, d=512, heads=8, kv_heads=2, hd=64, ffn=1024, vocab=256):
    """A Model.fused_ops() model of the given sizes without any weights: the checks read the sizes alone."""
    import torch
    w = lambda t, rows, cols: decode.DevWeight(None, t, rows, cols)  # noqa: E731
    m = decode.Model(lm_head=w(qvx.Q6_K, vocab, d), output_norm=torch.ones(d))
    for _ in range(layers):
        m.layers.append({"wqk": w(qvx.Q4_K, (heads + kv_heads) * hd, d), "wv": w(qvx.Q6_K, kv_heads * hd, d),
                         "wo": w(qvx.Q4_K, d, heads * hd), "ffn_gateup": w(qvx.Q4_K, 2 * ffn, d),
                         "ffn_down": w(qvx.Q6_K, d, ffn)})
        m.norms.append({"attn_norm": torch.ones(d), "ffn_norm": torch.ones(d)})
    return m


def _paged_step(model, **kw):
    a = dict(m=1, heads=8, kv_heads=2, n_pages=4, max_pages=2, device="meta")
    a.update(kw)
    return decode.PagedDecodeStep(model, **a)


def test_paged_step_refuses_projections_that_do_not_fit():
    """The step's buffers are sized once: a projection of any layer that would write or read past them, or whose heads
    are not where the rotation looks for them, is refused before anything is allocated."""
    import pytest

    with pytest.raises(ValueError, match="KvCache.of"):  # the sizes fit: it comes as far as the device's memory
        _paged_step(_paged_model())
    for layer in (0, 1):
        for key, rows, cols in (("wqk", 8 * 64, 512), ("wqk", 11 * 64, 512), ("wqk", 10 * 64, 256), ("wv", 4 * 64, 512),
                                ("wv", 2 * 64, 768), ("wo", 768, 512), ("wo", 512, 768), ("ffn_gateup", 4096, 512),
                                ("ffn_gateup", 2048, 768), ("ffn_down", 512, 2048), ("ffn_down", 768, 1024)):
            m = _paged_model()
            m.layers[layer][key] = decode.DevWeight(None, m.layers[layer][key].type, rows, cols)
            with pytest.raises(ValueError, match="PagedDecodeStep"):
                _paged_step(m)
        m = _paged_model()
        m.norms[layer]["attn_norm"] = m.norms[layer]["attn_norm"][:256]
        with pytest.raises(ValueError, match="PagedDecodeStep"):
            _paged_step(m)
    m = _paged_model()
    m.lm_head = decode.DevWeight(None, qvx.Q6_K, 256, 768)
    with pytest.raises(ValueError, match="PagedDecodeStep"):
        _paged_step(m)
    m = _paged_model()
    m.norms.pop()
    with pytest.raises(ValueError, match="norms of layer 1"):
        _paged_step(m)
    for kw in (dict(m=0), dict(heads=0), dict(kv_heads=0), dict(kv_heads=-2), dict(n_pages=0), dict(max_pages=0),
               dict(page_size=0)):
        with pytest.raises(ValueError, match="PagedDecodeStep"):
            _paged_step(_paged_model(), **kw)


def test_paged_step_refuses_a_head_without_its_norm():
    import pytest

    for norm in (None, "short"):
        m = _paged_model()
        m.output_norm = None if norm is None else m.output_norm[:256]
        with pytest.raises(ValueError, match="output_norm"):
            _paged_step(m)


def _gguf(arch="llama", **keys):
    from gguf_build import GgufBuilder
    from qorvix_amd.gguf import GgufFile
    b = GgufBuilder(3).str("general.architecture", arch)
    for key, value in keys.items():
        key = f"{arch}.rope.{key.replace('__', '.')}"
        b = b.str(key, value) if isinstance(value, str) else b.u32(key, value) if isinstance(value, int) else b.f32(key, value)
    return GgufFile.parse(b.build(32))


def test_rotation_of_a_file():
    """The pairing, base and scaling that the file's q and k rows were laid out for, not the synthetic model's."""
    r = decode.Rotation.of_gguf(_gguf(freq_base=500000.0, dimension_count=64))
    assert (r.base, r.dim, r.pairing, r.scaling, r.factors, r.magnitude) == (500000.0, 64, qvx.ROPE_PAIRS, 1.0, None, 1.0)
    assert decode.Rotation.of_gguf(_gguf()) == decode.Rotation(10000.0, qvx.ROPE_PAIRS)
    assert decode.Rotation.of_gguf(_gguf(scaling__type="linear", scaling__factor=4.0)).scaling == 4.0
    assert decode.Rotation.of_gguf(_gguf(scaling__type="none", scaling__factor=4.0)).scaling == 1.0
    assert decode.Rotation.of_gguf(_gguf(scale_linear=2.0)).scaling == 2.0
    assert decode.Rotation.of_gguf(_gguf(scaling__type="yarn", scaling__factor=4.0)).scaling is None
    assert decode.Rotation.of_gguf(_gguf("other")).pairing is None


def test_paged_step_takes_the_models_rotation():
    """Fused forms carry the rotation; one that a file leaves open, or that does not fit the heads, is refused unless the
    caller gives one."""
    import pytest

    def layers():
        m = decode.Model(rotation=decode.Rotation(pairing=qvx.ROPE_PAIRS))
        return m
    assert layers().fused().rotation.pairing == layers().fused_ops().rotation.pairing == qvx.ROPE_PAIRS
    for bad in (decode.Rotation(pairing=None), decode.Rotation(scaling=None), decode.Rotation(dim=72), decode.Rotation(dim=12)):
        m = _paged_model()
        m.rotation = bad
        with pytest.raises(ValueError, match="[Rr]otation"):
            _paged_step(m)
        with pytest.raises(ValueError, match="KvCache.of"):
            _paged_step(m, rotation=decode.Rotation(dim=32))


def test_rotation_frequencies():
    import torch
    r = decode.Rotation(base=100.0, dim=16, scaling=2.0, factors=torch.arange(1.0, 9.0))
    want = torch.tensor([100.0 ** (-i / 8) / 2 / (i + 1) for i in range(8)], dtype=torch.float64)
    assert torch.allclose(r.frequencies(32, "cpu"), want, rtol=1e-14, atol=0)
    assert decode.Rotation().frequencies(64, "cpu").shape == (32,) and decode.Rotation(dim=0).frequencies(64, "cpu").shape == (0,)


def test_paged_step_refuses_layers_with_more_than_it_computes():
    """A bias, a norm of q and k, another layer form in the file: the projections alone serve it, the whole step does not."""
    import pytest

    class File:
        tensors = [type("T", (), dict(name=n)) for n in (
            "token_embd.weight", "output.weight", "rope_freqs.weight", "blk.0.attn_q.weight", "blk.0.attn_q.bias",
            "blk.1.ffn_norm.weight", "blk.1.attn_q_norm.weight", "blk.0.ffn_down.weight", "position_embd.weight")]
    assert decode.Model.not_computed(File) == ["blk.0.attn_q.bias", "blk.1.attn_q_norm.weight"]
    m = _paged_model()
    m.left_out = decode.Model.not_computed(File)
    with pytest.raises(ValueError, match="blk.0.attn_q.bias"):
        _paged_step(m)
    assert decode.Model(left_out=["a"]).fused().left_out == decode.Model(left_out=["a"]).fused_ops().left_out == ["a"]


def test_a_files_rotation_never_keeps_its_weights_from_loading():
    """Divisors of another type than F32 leave the rotation open, for the step alone to refuse."""
    import pytest
    from gguf_build import GgufBuilder
    from qorvix_amd.gguf import GgufFile
    b = GgufBuilder(3).str("general.architecture", "llama")
    b.tensor("rope_freqs.weight", [8], qvx.F16, 0)
    r = decode.Rotation.of_gguf(GgufFile.parse(b.build(32, data=bytes(32))))
    assert r.scaling is None and r.factors is None
    for bad in (r, decode.Rotation(base=0.0), decode.Rotation(base=-1.0), decode.Rotation(scaling=0.0)):
        with pytest.raises(ValueError):
            bad.frequencies(64, "cpu")


def test_rotation_takes_one_divisor_for_all_pairs():
    """A caller's `rope_factors` of one value divide every pair, as they did before files had their own."""
    import torch
    want = decode.Rotation().frequencies(64, "cpu") / 4
    for factors in (torch.tensor(4.0), torch.tensor([4.0]), torch.full((32,), 4.0)):
        got = decode.Rotation(factors=factors).frequencies(64, "cpu")
        assert got.shape == (32,) and torch.equal(got, want)
