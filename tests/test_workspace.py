"""The scratch handed out per device: what a call gets depends on what it asks for, not on the calls before it (no GPU)."""
import torch

from apt_serve_b200 import _native as N
from apt_serve_b200 import attention as A

CPU = torch.device("cpu")
SHAPE = (64, 40, 16, 40, 128)


def test_scratch_size_does_not_depend_on_earlier_calls(monkeypatch):
    """A layer-step re-projects or attends directly by the size of its scratch: an attention-sized one must not have
    grown with someone else's layer-step."""
    monkeypatch.setattr(A, "_workspaces", {})
    plain = N.lib().aps_attention_workspace_bytes(*SHAPE)
    step = N.lib().aps_decode_layer_step_workspace_bytes(*SHAPE, 5120, N.DTYPE_ENUM[torch.float16])
    assert 1 << 20 < plain < step
    assert A.attention_workspace(CPU, *SHAPE).numel() == plain
    big = A.layer_step_workspace(CPU, *SHAPE, 5120, torch.float16)
    assert big.numel() == step
    again = A.attention_workspace(CPU, *SHAPE)
    assert again.numel() == plain and again.data_ptr() == big.data_ptr()
    assert A.attention_workspace(CPU, 1, 1, 16, 1, 32).numel() == 1 << 20
    assert A.layer_step_workspace(CPU, *SHAPE, 5120, torch.float16).data_ptr() == big.data_ptr()


def test_scratch_of_a_few_requests_is_small():
    """The projected outputs and the partial scores are sized for the batch, not for a full group of requests."""
    size = lambda b, blocks, t: N.lib().aps_decode_layer_step_workspace_bytes(b, blocks, 16, 40, 128, 5120, N.DTYPE_ENUM[t])
    one = size(1, 39, torch.float16)
    # 16 requests' folded queries in two terms, seven ranges of projected outputs, partial scores of 3 tiles and 51 pieces,
    # 39 blocks of weights, the plan and some rounding
    assert one < 16 * (2 * 40 * 5120 * 2 + 7 * 5120 * 4) + (3 + 51) * 40 * 1024 + 39 * 2 * 48 * 32 + (1 << 18)
    assert size(8, 39, torch.float16) < 2 * one and size(256, 128, torch.float16) > 10 * one
    small = N.lib().aps_decode_layer_step_workspace_bytes(1, 39, 16, 12, 64, 768, N.DTYPE_ENUM[torch.float32])
    assert small < 4 << 20


def test_scratch_of_captured_calls_is_kept(monkeypatch):
    """A graph goes on working in it after a call that needs more."""
    monkeypatch.setattr(A, "_workspaces", {})
    monkeypatch.setattr(A, "_captured", {})
    monkeypatch.setattr(A, "_outgrown", [])
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device, **kw: empty(*a, **kw))
    device = torch.device("cuda", 0)
    A._scratch_of(device, 2 << 20)
    A._scratch_of(device, 3 << 20)
    assert A._outgrown == []      # no graph knew it
    capturing[0] = True
    first = A._scratch_of(device, 1 << 20)[0]
    assert first.numel() == 3 << 20
    capturing[0] = False
    assert A._scratch_of(device, 2 << 20)[0] is first
    second = A._scratch_of(device, 4 << 20)[0]
    third = A._scratch_of(device, 5 << 20)[0]
    assert len(A._outgrown) == 1 and A._outgrown[0] is first and third is not second
    capturing[0] = True
    fourth = A._scratch_of(device, 6 << 20)[0]   # allocated under capture
    capturing[0] = False
    A._scratch_of(device, 7 << 20)
    assert len(A._outgrown) == 2 and A._outgrown[1] is fourth
