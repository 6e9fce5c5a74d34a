"""LlamaWeights.from_gguf refuses a head that a decode step cannot run, by name and before anything is loaded."""
import pytest
import torch

import gguf_writer as W
from inference_amd import QmmError, qmm
from inference_amd.llama_decode import LlamaWeights

H, F, VOCAB = 256, 512, 64
BLOCK = {0: (1, 4), 12: (256, 144), 14: (256, 210), 39: (32, 17)}


def image(embed_type, head_type):
    meta = [("general.architecture", W.T_STRING, "llama"), ("llama.block_count", W.T_UINT32, 1),
            ("llama.embedding_length", W.T_UINT32, H), ("llama.feed_forward_length", W.T_UINT32, F),
            ("llama.attention.head_count", W.T_UINT32, 4), ("llama.attention.head_count_kv", W.T_UINT32, 2)]

    def t(name, shape, kind):
        n = 1
        for d in shape:
            n *= d
        return name, shape, kind, bytes(n // BLOCK[kind][0] * BLOCK[kind][1])

    ts = [t("token_embd.weight", (VOCAB, H), embed_type), t("output_norm.weight", (H,), 0),
          t("blk.0.attn_norm.weight", (H,), 0), t("blk.0.ffn_norm.weight", (H,), 0)]
    ts += [t(f"blk.0.{n}.weight", s, 12) for n, s in (
        ("attn_q", (H, H)), ("attn_k", (H // 2, H)), ("attn_v", (H // 2, H)), ("attn_output", (H, H)),
        ("ffn_gate", (F, H)), ("ffn_up", (F, H)), ("ffn_down", (H, F)))]
    if head_type is not None:
        ts.append(t("output.weight", (VOCAB, H), head_type))
    return W.build(meta, ts)


@pytest.mark.parametrize("embed,head,name", [(12, 39, "output.weight"), (0, 39, "output.weight"),
                                             (39, None, "token_embd.weight")])
def test_mxfp4_heads_are_refused(tmp_path, embed, head, name):
    p = tmp_path / "m.gguf"
    p.write_bytes(image(embed, head))
    with pytest.raises(QmmError, match=f"{name} has GGML type 39") as e:
        LlamaWeights.from_gguf(p, torch.device("cuda:0"))
    assert e.value.status == qmm.QMM_ERR_UNSUPPORTED


@pytest.mark.gpu
@pytest.mark.parametrize("embed,head", [(39, 14), (12, None), (14, 12)])
def test_other_heads_load(tmp_path, embed, head):
    p = tmp_path / "m.gguf"
    p.write_bytes(image(embed, head))
    w = LlamaWeights.from_gguf(p, torch.device("cuda:0"))
    assert int(w.head.dtype()) == (head or embed) and w.embed.shape == (VOCAB, H)
