"""residual_out beside the inputs' memory: in their place, value for value, or apart (CPU tensors, the launch stubbed)."""
import pytest
import torch

from test_lora_norm_args import Launched, ops  # noqa: F401

BF16 = torch.bfloat16


@pytest.mark.parametrize("fp8", [False, True])
def test_residual_out_overlaps(ops, fp8):  # noqa: F811
    M, H = 6, 256
    fn = ops.add_rms_norm_fp8 if fp8 else ops.add_rms_norm
    buf = torch.zeros(4 * M * H, dtype=BF16)
    rows = lambda at: buf[at * H:(at + M) * H].view(M, H)  # noqa: E731
    x, w = torch.zeros(M, H, dtype=BF16), torch.zeros(H, dtype=BF16)
    good = dict(x=x, residual=rows(0), weight=w, eps=1e-6)

    def taken(**kw):
        with pytest.raises(Launched):
            fn(**{**good, **kw})

    def refused(name, **kw):
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            fn(**{**good, **kw})

    taken(residual_out=rows(0))
    taken(residual_out=rows(M))
    taken(x=rows(M), residual_out=rows(M))
    taken(x=rows(M), residual=None, residual_out=rows(M))
    taken(gate=rows(M), residual_out=rows(M))
    taken(x=rows(0), residual=rows(0), gate=rows(0), residual_out=rows(0))
    for at in (1, M - 1):
        refused("residual", residual_out=rows(at))
        refused("residual", residual=rows(at), residual_out=rows(0))
        refused("x", x=rows(M), residual=x, residual_out=rows(M + at))
        refused("gate", gate=rows(M), residual_out=rows(M + at))
    # rows of a wider buffer, columns, a gate per row, weights, an fp32 stream over bf16 rows
    refused("residual", residual=buf[:2 * M * H].view(M, 2 * H)[:, :H], residual_out=rows(0))
    refused("gate", gate=buf[:H], residual_out=rows(0), residual=x)
    refused("gate", gate=buf[:M].view(M, 1), residual_out=rows(0), residual=x)
    refused("weight", weight=buf[H:2 * H], residual_out=rows(0), residual=x)
    refused("post_weight", post_weight=buf[:H], residual_out=rows(0), residual=x)
    wide = torch.zeros(M, H)
    refused("x", x=wide.view(BF16).view(2 * M, H)[:M], residual=torch.zeros(M, H), residual_out=wide)
    # one row is a row wherever its neighbours are; no rows are none
    fn_one = dict(x=x[:1], weight=w, eps=1e-6)
    with pytest.raises(Launched):
        fn(residual=buf[:2 * H].view(1, 2 * H)[:, :H], residual_out=rows(0)[:1], **fn_one)
    with pytest.raises(Launched):
        fn(x=x[:0], residual=rows(0)[:0], weight=w, eps=1e-6, residual_out=rows(1)[:0])


@pytest.mark.parametrize("fp8", [False, True])
def test_one_row_over_its_weights(ops, fp8):  # noqa: F811
    """The weights are read behind the store of the stream: a single row's are not its output's place either."""
    H = 256
    fn = ops.add_rms_norm_fp8 if fp8 else ops.add_rms_norm
    buf, x = torch.zeros(1, H, dtype=BF16), torch.zeros(1, H, dtype=BF16)
    good = dict(x=x, residual=x, weight=x[0].clone(), eps=1e-6, post_weight=x[0].clone(), residual_out=buf)
    for name in ("weight", "post_weight"):
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            fn(**{**good, name: buf[0]})
    with pytest.raises(Launched):
        fn(**{**good, "gate": buf[0]})
