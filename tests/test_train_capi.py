"""The token-network entry points without a GPU: argument checks on the host, workspace sizes, and
the store-data hazard of their kernels' assembly."""
import subprocess

import pytest
import torch

import my_own_cnn_amd as M
from my_own_cnn_amd import _capi
from my_own_cnn_amd import build as B
from tests.test_isa_store_gaps import store_gaps

P = 4096  # an address that no refused call reads
BIG = 1 << 62
NULL, BAD, UNSUPPORTED = _capi.MIQ_ERR_NULL_POINTER, _capi.MIQ_ERR_INVALID_ARGUMENT, _capi.MIQ_ERR_UNSUPPORTED


def _call(entry, defaults, **change):
    args = dict(defaults, **change)
    status = getattr(M.lib(), entry)(*args.values())
    return status, M.lib().miq_last_error_message().decode()


FPROP = dict(table=P, ids=P, y=P, vocab=10, c=8, tokens=4, ld_table=8, ld_y=8, scale=1.0, table_type=0, id_type=3,
             y_type=0, stream=None)
GRAD = dict(dy=P, ids=P, dtable=P, vocab=10, c=8, tokens=4, ld_dy=8, ld_dtable=8, scale=1.0, accumulate=0, dy_type=0,
            id_type=3, dtable_type=0, ws=P, ws_bytes=BIG, stream=None)
ACT = dict(x=P, y=P, codes=P, scales=P, rows=4, c=8, ld_x=8, ld_y=8, act=2, gated=0, type=0, stream=None)
BACK = dict(dy=P, codes=P, scales=P, dx=P, rows=4, c=8, ld_dy=8, ld_dx=8, act=2, gated=0, type=0, stream=None)
EXPAND = dict(codes=P, scales=P, y=P, rows=4, c=8, ld_y=8, act=0, gated=0, type=0, stream=None)
WGRAD = dict(dy=P, codes=P, scales=P, dw=P, rows=4, c=8, k=8, ld_dy=8, ld_dw=8, accumulate=0, dy_type=0, dw_type=0,
             ws=P, ws_bytes=BIG, stream=None)

REFUSED = [
    ("miq_embed_fprop", FPROP, dict(vocab=-1), BAD, ">= 0"),
    ("miq_embed_fprop", FPROP, dict(vocab=(1 << 28) + 1), BAD, "2^28"),
    ("miq_embed_fprop", FPROP, dict(tokens=1 << 31), BAD, "2^31 - 65"),
    ("miq_embed_fprop", FPROP, dict(c=(1 << 29) + 1), BAD, "2^29"),
    ("miq_embed_fprop", FPROP, dict(ld_table=7), BAD, "row distance"),
    ("miq_embed_fprop", FPROP, dict(ld_y=7), BAD, "row distance"),
    ("miq_embed_fprop", FPROP, dict(table_type=2), BAD, "table_type"),
    ("miq_embed_fprop", FPROP, dict(id_type=0), BAD, "id_type"),
    ("miq_embed_fprop", FPROP, dict(y_type=9), BAD, "y_type"),
    ("miq_embed_fprop", FPROP, dict(ids=None), NULL, "ids"),
    ("miq_embed_fprop", FPROP, dict(y=None), NULL, "output"),
    ("miq_embed_fprop", FPROP, dict(table=None), NULL, "table"),
    ("miq_embed_fprop", FPROP, dict(table=P + 2), BAD, "aligned"),
    ("miq_embed_fprop", FPROP, dict(ids=P + 4), BAD, "aligned"),
    ("miq_embed_grad", GRAD, dict(tokens=-1), BAD, ">= 0"),
    ("miq_embed_grad", GRAD, dict(accumulate=2), BAD, "accumulate"),
    ("miq_embed_grad", GRAD, dict(dy_type=3), BAD, "dy_type"),
    ("miq_embed_grad", GRAD, dict(ld_dy=7), BAD, "row distance"),
    ("miq_embed_grad", GRAD, dict(dtable=None), NULL, "output"),
    ("miq_embed_grad", GRAD, dict(dy=None), NULL, "dy"),
    ("miq_embed_grad", GRAD, dict(tokens=2000, ws=None), NULL, "workspace"),
    ("miq_embed_grad", GRAD, dict(tokens=2000, ws_bytes=8), BAD, "workspace is smaller"),
    ("miq_embed_grad", GRAD, dict(ws=P + 8), BAD, "16 bytes"),
    ("miq_act8_fprop", ACT, dict(rows=-1), BAD, ">= 0"),
    ("miq_act8_fprop", ACT, dict(rows=1 << 41), BAD, "2^40"),
    ("miq_act8_fprop", ACT, dict(rows=1 << 39, c=1 << 20, ld_x=1 << 20, ld_y=1 << 20), BAD, "2^46"),
    ("miq_act8_fprop", ACT, dict(act=4), BAD, "act must be"),
    ("miq_act8_fprop", ACT, dict(gated=2), BAD, "gated"),
    ("miq_act8_fprop", ACT, dict(gated=1), BAD, "row distance"),
    ("miq_act8_fprop", ACT, dict(type=2), BAD, "type must be"),
    ("miq_act8_fprop", ACT, dict(x=None), NULL, "input"),
    ("miq_act8_fprop", ACT, dict(codes=None), NULL, "codes"),
    ("miq_act8_fprop", ACT, dict(scales=None), NULL, "scales"),
    ("miq_act8_fprop", ACT, dict(x=P + 1, type=1), BAD, "aligned"),
    ("miq_act8_bprop", BACK, dict(dy=None), NULL, "dy"),
    ("miq_act8_bprop", BACK, dict(dx=None), NULL, "output"),
    ("miq_act8_bprop", BACK, dict(gated=1, ld_dx=15), BAD, "row distance"),
    ("miq_act8_bprop", BACK, dict(act=-1), BAD, "act must be"),
    ("miq_act8_expand", EXPAND, dict(y=None), NULL, "output"),
    ("miq_act8_expand", EXPAND, dict(codes=None), NULL, "codes"),
    ("miq_act8_expand", EXPAND, dict(ld_y=3), BAD, "row distance"),
    ("miq_act8_grad", WGRAD, dict(rows=1 << 31), BAD, "2^31 - 65"),
    ("miq_act8_grad", WGRAD, dict(c=1 << 23), BAD, "2^22"),
    ("miq_act8_grad", WGRAD, dict(c=1 << 22, k=1 << 22, ld_dy=1 << 22, ld_dw=1 << 22), UNSUPPORTED, "2^23"),
    ("miq_act8_grad", WGRAD, dict(dw_type=1), BAD, "dw_type"),
    ("miq_act8_grad", WGRAD, dict(dy_type=2), BAD, "dy_type"),
    ("miq_act8_grad", WGRAD, dict(accumulate=-1), BAD, "accumulate"),
    ("miq_act8_grad", WGRAD, dict(ld_dw=7), BAD, "row distance"),
    ("miq_act8_grad", WGRAD, dict(dw=None), NULL, "output"),
    ("miq_act8_grad", WGRAD, dict(codes=None), NULL, "codes"),
    ("miq_act8_grad", WGRAD, dict(rows=100000, ws=None), NULL, "workspace"),
    ("miq_act8_grad", WGRAD, dict(rows=100000, ws_bytes=8), BAD, "workspace is smaller"),
]


@pytest.mark.parametrize("entry,defaults,change,status,text", REFUSED,
                         ids=["{}-{}".format(r[0][4:], "-".join(r[2])) + str(i) for i, r in enumerate(REFUSED)])
def test_refused_before_anything_runs(entry, defaults, change, status, text):
    got, message = _call(entry, defaults, **change)
    assert got == status and text in message


@pytest.mark.parametrize("entry,defaults,change", [
    ("miq_embed_fprop", FPROP, dict(tokens=0, ids=None, y=None)),
    ("miq_embed_fprop", FPROP, dict(c=0, y=None)),
    ("miq_embed_grad", GRAD, dict(vocab=0, dtable=None)),
    ("miq_embed_grad", GRAD, dict(tokens=0, accumulate=1, dtable=None, dy=None)),
    ("miq_act8_fprop", ACT, dict(rows=0, x=None, y=None, codes=None)),
    ("miq_act8_bprop", BACK, dict(c=0, dy=None)),
    ("miq_act8_expand", EXPAND, dict(rows=0, y=None)),
    ("miq_act8_grad", WGRAD, dict(k=0, dw=None)),
    ("miq_act8_grad", WGRAD, dict(rows=0, accumulate=1, dw=None)),
])
def test_nothing_to_do_enqueues_nothing(entry, defaults, change):
    assert _call(entry, defaults, **change)[0] == _capi.MIQ_OK


def test_workspace_sizes():
    assert M.embed_grad_workspace_size(1000, 64, 0) == 0
    assert M.embed_grad_workspace_size(1000, 64, 1024) == 0  # few tokens are not sorted
    small, large = M.embed_grad_workspace_size(1000, 64, 1025), M.embed_grad_workspace_size(1000, 64, 10 ** 6)
    assert 0 < small < large < 10 ** 6 * 16 + (64 << 20)
    assert M.embed_grad_workspace_size(1 << 28, 1 << 20, (1 << 31) - 65) > 0
    assert M.act8_grad_workspace_size(64, 4096, 4096) == 0
    assert 0 < M.act8_grad_workspace_size(10 ** 6, 128, 128, torch.bfloat16) <= 64 << 20
    with pytest.raises(M.MiqError, match=">= 0"):
        M.embed_grad_workspace_size(-1, 64, 0)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        M.act8_grad_workspace_size(64, 64, 64, torch.float16)
    assert M.lib().miq_embed_grad_workspace_size(1, 1, 1, None) == NULL
    assert M.lib().miq_act8_grad_workspace_size(1, 1, 1, 0, None) == NULL


def test_weight_gradient_plan():
    assert M.plan_act8_grad(512, 1024, 1024, torch.bfloat16) == (64, 1)
    assert M.plan_act8_grad(16384, 4096, 4096, torch.bfloat16) == (256, 1)
    assert M.plan_act8_grad(0, 64, 64) == (64, 1) and M.plan_act8_grad(64, 0, 64) == (0, 0)
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (1, 31, 65, 1000, 12345, 10 ** 6):
            for c in (1, 200, 3000):
                for k in (5, 64, 2000):
                    tile, splits = M.plan_act8_grad(rows, c, k, dtype)
                    assert tile in (64, 128, 256) and 1 <= splits <= max(1, rows // 32)
                    bytes_ = M.act8_grad_workspace_size(rows, c, k, dtype)
                    assert bytes_ == (splits * c * k * 4 if splits > 1 else 0)
    with pytest.raises(M.MiqError, match="2\\^22"):
        M.plan_act8_grad(1, 1 << 23, 1)
    assert M.lib().miq_plan_act8_grad(1, 1, 1, 0, None) == NULL


def test_host_tensors_are_refused():
    x, ids = torch.zeros((3, 8)), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: M.embed_fprop(x, ids), lambda: M.embed_grad(x, ids, 4), lambda: M.act8_keep(x),
                 lambda: M.act8_grad(x, M.Act8(x.to(torch.int8), x[:, :1].to(torch.uint8).contiguous()))):
        with pytest.raises(ValueError, match="device memory"):
            call()


@pytest.mark.parametrize("src", ["embed.hip", "embed_grad.hip", "act8.hip", "act8_grad.hip"])
def test_every_wide_store_is_followed_by_two_wait_states(src, tmp_path):
    dst = tmp_path / "k.s"
    subprocess.run([B.hipcc(), *B.common_flags(), "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(dst)],
                   check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    short = [g for g in store_gaps(dst.read_text().splitlines()) if g[3] < 2]
    assert not short, short[:5]


