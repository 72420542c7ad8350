"""Gates that mask the groups that are not kept with 0, and with -inf: what becomes of their choice when the bias turns negative."""
import pytest
import torch

from moelab_amd import patch
from test_patch import D
from test_patch_scored import settings, sigmoid_block


def masks_with(value, block):
    """DeepSeek-V3's gate in plain steps, the other groups' experts at `value`."""
    class Gate(type(block.gate)):
        def forward(self, x):
            logits = torch.nn.functional.linear(x.reshape(-1, D).float(), self.weight.float())
            s = torch.sigmoid(logits)
            c = (s + self.e_score_correction_bias).reshape(len(s), 4, 4)
            kept = c.topk(2, dim=-1).values.sum(-1).topk(2, dim=-1).indices
            mask = torch.zeros(len(s), 4, dtype=torch.bool, device=s.device).scatter(1, kept, True)
            idx = torch.where(mask[..., None], c, value).flatten(1).topk(4, dim=-1).indices
            w = s.gather(1, idx)
            return logits, 2.5 * w / w.sum(-1, keepdim=True), idx
    block.gate.__class__ = Gate
    return block


def test_which_masks():
    assert settings(masks_with(0.0, sigmoid_block("cpu"))) is None
    want = settings(sigmoid_block("cpu"))
    assert want is not None and settings(masks_with(-float("inf"), sigmoid_block("cpu"))) == want
    cfg = patch.block_state(masks_with(0.0, sigmoid_block("cpu")))
    assert cfg["kind"] == "deepseek" and cfg["stock_gate"] and cfg["scored"] is None


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [0.0, -float("inf")])
def test_a_bias_that_turns_negative_unseen(mask):
    """Through .data, which no version counts, and under a captured graph: the patched block chooses as its gate does."""
    from helpers import assert_close
    block = masks_with(mask, sigmoid_block("cuda"))
    x = torch.randn(1, 24, D, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    patch.patch_block(block)
    block.float()
    patch.load_dequantised(block)
    block.gate.weight.data = block.gate.weight.data.to(torch.bfloat16)
    bias = block.gate.e_score_correction_bias
    with torch.no_grad():
        block(x)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            y = block(x)
        for _ in range(3):
            bias.data.sub_(0.7)
            flat = x.reshape(-1, D).float()
            out = block.gate(flat)
            ref = block.experts(flat, out[2].long(), out[1].float()) + block.shared_experts(flat)
            graph.replay()
            torch.cuda.synchronize()
            for got in (y.clone(), block(x)):
                assert_close(got.reshape(-1, D), ref.cpu().numpy(), what=("masked with", mask))
