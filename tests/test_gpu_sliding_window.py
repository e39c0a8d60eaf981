"""A file whose layers see a window, from its bytes to decode.PagedDecodeStep.  Reference and tolerance as in
test_gpu_shared_serving.py."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx
from qorvix_amd import decode
from test_gpu_shared_serving import HostShared, _both

pytestmark = pytest.mark.gpu


def test_a_file_with_a_window(cuda, tmp_path):
    from gguf_build import GgufBuilder
    torch = cuda
    rng = np.random.default_rng(9)
    d, heads, kv_heads, hd, ffn = 512, 8, 2, 64, 512
    b = (GgufBuilder(3).str("general.architecture", "llama").u32("general.alignment", 32).u32("llama.block_count", 1)
         .u32("llama.embedding_length", d).u32("llama.feed_forward_length", ffn).u32("llama.attention.head_count", heads)
         .u32("llama.attention.head_count_kv", kv_heads).u32("llama.attention.sliding_window", 5))
    tensors = [(n, [d], (1.0 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for n in
               ("blk.0.attn_norm.weight", "blk.0.ffn_norm.weight", "output_norm.weight")]
    tensors += [(f"blk.0.{n}.weight", [cols, rows], (rng.standard_normal((rows, cols)) * cols ** -0.5).astype(np.float32))
                for n, rows, cols in (("attn_q", d, d), ("attn_k", kv_heads * hd, d), ("attn_v", kv_heads * hd, d),
                                      ("attn_output", d, d), ("ffn_gate", ffn, d), ("ffn_up", ffn, d), ("ffn_down", d, ffn))]
    tensors.append(("token_embd.weight", [d, 64], rng.standard_normal((64, d)).astype(np.float32)))
    data = bytearray()
    for name, dims, x in tensors:
        b.tensor(name, dims, qvx.F32, len(data))
        data += x.tobytes()
    path = tmp_path / "model.gguf"
    path.write_bytes(b.build(32, data=bytes(data)))
    model = decode.Model.from_gguf(path).fused_ops()
    make = lambda **kw: decode.PagedDecodeStep(model, 2, heads, kv_heads, n_pages=8, max_pages=3, page_size=4,  # noqa: E731
                                               rotation=decode.Rotation(), **kw)
    with pytest.raises(ValueError, match="see 5 tokens, the table holds 12"):
        make()
    for window in (5, 12):  # the file's, and full attention
        step = make(window=window)
        _both(torch, step, HostShared(torch, step, torch.float16, window), 9)
