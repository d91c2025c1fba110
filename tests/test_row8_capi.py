"""The entry points of the norm and of 8-bit rows without a GPU: argument checks on the host, workspace
sizes, and the store-data hazard of their kernels' assembly."""
import subprocess

import pytest
import torch

import my_own_cnn_amd as M
from my_own_cnn_amd import _capi
from my_own_cnn_amd import build as B
from tests.test_isa_store_gaps import store_gaps
from tests.test_train_capi import BAD, BIG, NULL, P, _call

NORM = dict(x=P, add=P, gain=P, sum=P, y=P, rows=4, c=8, ld_x=8, ld_add=8, ld_sum=8, ld_y=8, eps=1e-6, type=0,
            gain_type=0, stream=None)
NORM8 = dict(x=P, add=P, gain=P, sum=P, codes=P, scales=P, rows=4, c=8, ld_x=8, ld_add=8, ld_sum=8, eps=1e-6, type=0,
             gain_type=0, stream=None)
BACK = dict(dy=P, x=P, gain=P, dsum=P, dx=P, dgain=P, rows=4, c=8, ld_dy=8, ld_x=8, ld_dsum=8, ld_dx=8, eps=1e-6,
            accumulate=0, type=0, gain_type=0, dgain_type=0, ws=P, ws_bytes=BIG, stream=None)
ACT = dict(x=P, codes=P, scales=P, rows=4, c=8, ld_x=8, act=2, gated=0, type=0, stream=None)
EXPAND = dict(codes=P, scales=P, y=P, rows=4, c=8, ld_y=8, type=0, stream=None)
LINEAR = dict(codes=P, scales=P, w_codes=P, w_scales=P, bias=P, add=P, y=P, rows=4, c=8, k=8, ld_add=8, ld_y=8, type=0,
              ws=P, ws_bytes=BIG, stream=None)
EXPERTS = dict(codes=P, scales=P, w_codes=P, w_scales=P, bias=P, offsets=P, index=P, y=P, x_rows=4, rows=4, c=8, k=8,
               experts=2, ld_y=8, type=0, ws=P, ws_bytes=BIG, stream=None)
PLAN = dict(ids=P, offsets=P, rows=P, places=P, tokens=4, slots=2, experts=3, id_type=2, stream=None)
JOIN = dict(y=P, places=P, share=P, add=P, out=P, rows=4, tokens=4, slots=2, c=8, ld_y=8, ld_add=8, ld_out=8, type=0,
            stream=None)

REFUSED = [
    ("miq_rms_fprop", NORM, dict(rows=-1), BAD, ">= 0"),
    ("miq_rms_fprop", NORM, dict(rows=1 << 41), BAD, "2^40"),
    ("miq_rms_fprop", NORM, dict(c=(1 << 29) + 1), BAD, "2^29"),
    ("miq_rms_fprop", NORM, dict(eps=0.0), BAD, "eps"),
    ("miq_rms_fprop", NORM, dict(eps=float("nan")), BAD, "eps"),
    ("miq_rms_fprop", NORM, dict(eps=float("inf")), BAD, "eps"),
    ("miq_rms_fprop", NORM, dict(type=2), BAD, "type"),
    ("miq_rms_fprop", NORM, dict(gain_type=3), BAD, "gain_type"),
    ("miq_rms_fprop", NORM, dict(ld_x=7), BAD, "row distance"),
    ("miq_rms_fprop", NORM, dict(ld_add=7), BAD, "row distance"),
    ("miq_rms_fprop", NORM, dict(ld_sum=7), BAD, "row distance"),
    ("miq_rms_fprop", NORM, dict(ld_y=7), BAD, "row distance"),
    ("miq_rms_fprop", NORM, dict(x=None), NULL, "input"),
    ("miq_rms_fprop", NORM, dict(gain=None), NULL, "gain"),
    ("miq_rms_fprop", NORM, dict(sum=None), NULL, "come together"),
    ("miq_rms_fprop", NORM, dict(add=None), NULL, "come together"),
    ("miq_rms_fprop", NORM, dict(y=None), NULL, "output"),
    ("miq_rms_fprop", NORM, dict(x=P + 2), BAD, "aligned"),
    ("miq_rms_fprop", NORM, dict(gain=P + 1, gain_type=1), BAD, "aligned"),
    ("miq_rms_row8", NORM8, dict(codes=None), NULL, "output"),
    ("miq_rms_row8", NORM8, dict(scales=None), NULL, "output"),
    ("miq_rms_row8", NORM8, dict(scales=P + 2), BAD, "aligned"),
    ("miq_rms_row8", NORM8, dict(eps=-1.0), BAD, "eps"),
    ("miq_rms_bprop", BACK, dict(accumulate=2), BAD, "accumulate"),
    ("miq_rms_bprop", BACK, dict(dgain_type=2), BAD, "dgain_type"),
    ("miq_rms_bprop", BACK, dict(ld_dsum=7), BAD, "row distance"),
    ("miq_rms_bprop", BACK, dict(ld_dx=7), BAD, "row distance"),
    ("miq_rms_bprop", BACK, dict(dgain=None), NULL, "dgain"),
    ("miq_rms_bprop", BACK, dict(rows=0, dgain=None), NULL, "dgain"),
    ("miq_rms_bprop", BACK, dict(dy=None), NULL, "dy"),
    ("miq_rms_bprop", BACK, dict(dx=None), NULL, "output"),
    ("miq_rms_bprop", BACK, dict(ws=None), NULL, "workspace"),
    ("miq_rms_bprop", BACK, dict(ws_bytes=8), BAD, "workspace is smaller"),
    ("miq_rms_bprop", BACK, dict(ws=P + 8), BAD, "16 bytes"),
    ("miq_act_row8", ACT, dict(rows=-1), BAD, ">= 0"),
    ("miq_act_row8", ACT, dict(rows=1 << 39, c=1 << 20, ld_x=1 << 20), BAD, "2^46"),
    ("miq_act_row8", ACT, dict(act=4), BAD, "act must be"),
    ("miq_act_row8", ACT, dict(gated=2), BAD, "gated"),
    ("miq_act_row8", ACT, dict(gated=1), BAD, "row distance"),
    ("miq_act_row8", ACT, dict(type=2), BAD, "type"),
    ("miq_act_row8", ACT, dict(x=None), NULL, "input"),
    ("miq_act_row8", ACT, dict(codes=None), NULL, "codes"),
    ("miq_act_row8", ACT, dict(c=0, scales=None), NULL, "scales"),
    ("miq_row8_expand", EXPAND, dict(codes=None), NULL, "codes"),
    ("miq_row8_expand", EXPAND, dict(y=None), NULL, "output"),
    ("miq_row8_expand", EXPAND, dict(ld_y=3), BAD, "row distance"),
    ("miq_row8_expand", EXPAND, dict(type=3), BAD, "type"),
    ("miq_row8_linear", LINEAR, dict(rows=1 << 31), BAD, "2^31 - 65"),
    ("miq_row8_linear", LINEAR, dict(c=131072), BAD, "131071"),
    ("miq_row8_linear", LINEAR, dict(k=(1 << 22) + 1), BAD, "2^22"),
    ("miq_row8_linear", LINEAR, dict(k=-1), BAD, ">= 0"),
    ("miq_row8_linear", LINEAR, dict(ld_y=7), BAD, "row distance"),
    ("miq_row8_linear", LINEAR, dict(ld_add=7), BAD, "row distance"),
    ("miq_row8_linear", LINEAR, dict(type=2), BAD, "type"),
    ("miq_row8_linear", LINEAR, dict(codes=None), NULL, "codes"),
    ("miq_row8_linear", LINEAR, dict(w_scales=None), NULL, "scales"),
    ("miq_row8_linear", LINEAR, dict(y=None), NULL, "output"),
    ("miq_row8_linear", LINEAR, dict(bias=P + 2), BAD, "aligned"),
    ("miq_row8_linear", LINEAR, dict(add=P + 1, type=1), BAD, "aligned"),
    ("miq_row8_linear", LINEAR, dict(ws=P + 8), BAD, "16 bytes"),
    ("miq_row8_linear", LINEAR, dict(rows=8192, c=2001, k=4096, ld_add=4096, ld_y=4096, ws=None), NULL, "workspace"),
    ("miq_row8_linear", LINEAR, dict(rows=8192, c=2001, k=4096, ld_add=4096, ld_y=4096, ws_bytes=8), BAD, "smaller"),
    ("miq_row8_experts", EXPERTS, dict(rows=8192, x_rows=8192, c=2001, k=4096, ld_y=4096, ws=None), NULL, "workspace"),
    ("miq_row8_experts", EXPERTS, dict(rows=8192, x_rows=8192, c=2001, k=4096, ld_y=4096, ws_bytes=8), BAD, "smaller"),
    ("miq_row8_experts", EXPERTS, dict(ws=P + 4), BAD, "16 bytes"),
    ("miq_row8_experts", EXPERTS, dict(experts=0), BAD, "4096"),
    ("miq_row8_experts", EXPERTS, dict(experts=4097), BAD, "4096"),
    ("miq_row8_experts", EXPERTS, dict(x_rows=-1), BAD, "x_rows"),
    ("miq_row8_experts", EXPERTS, dict(x_rows=3, index=None), BAD, "as many rows"),
    ("miq_row8_experts", EXPERTS, dict(rows=1 << 31), BAD, "2^31 - 65"),
    ("miq_row8_experts", EXPERTS, dict(ld_y=7), BAD, "row distance"),
    ("miq_row8_experts", EXPERTS, dict(offsets=None), NULL, "offsets"),
    ("miq_row8_experts", EXPERTS, dict(scales=None), NULL, "scales"),
    ("miq_row8_experts", EXPERTS, dict(w_codes=None), NULL, "codes"),
    ("miq_row8_experts", EXPERTS, dict(y=None), NULL, "output"),
    ("miq_row8_experts", EXPERTS, dict(index=P + 1), BAD, "aligned"),
    ("miq_experts_plan", PLAN, dict(slots=0), BAD, "slots"),
    ("miq_experts_plan", PLAN, dict(tokens=-1), BAD, "tokens"),
    ("miq_experts_plan", PLAN, dict(tokens=1 << 30, slots=2), BAD, "2^31 - 65"),
    ("miq_experts_plan", PLAN, dict(experts=4097), BAD, "4096"),
    ("miq_experts_plan", PLAN, dict(id_type=0), BAD, "id_type"),
    ("miq_experts_plan", PLAN, dict(ids=None), NULL, "ids"),
    ("miq_experts_plan", PLAN, dict(offsets=None), NULL, "offsets"),
    ("miq_experts_plan", PLAN, dict(places=None), NULL, "output"),
    ("miq_experts_plan", PLAN, dict(ids=P + 4, id_type=3), BAD, "aligned"),
    ("miq_experts_join", JOIN, dict(rows=-1), BAD, "rows"),
    ("miq_experts_join", JOIN, dict(slots=0), BAD, "slots"),
    ("miq_experts_join", JOIN, dict(ld_add=7), BAD, "row distance"),
    ("miq_experts_join", JOIN, dict(type=2), BAD, "type"),
    ("miq_experts_join", JOIN, dict(y=None), NULL, "input"),
    ("miq_experts_join", JOIN, dict(places=None), NULL, "places"),
    ("miq_experts_join", JOIN, dict(out=None), NULL, "output"),
    ("miq_experts_join", JOIN, dict(share=P + 2), BAD, "aligned"),
]


@pytest.mark.parametrize("entry,defaults,change,status,text", REFUSED,
                         ids=["{}-{}".format(r[0][4:], "-".join(r[2])) + str(i) for i, r in enumerate(REFUSED)])
def test_refused_before_anything_runs(entry, defaults, change, status, text):
    got, message = _call(entry, defaults, **change)
    assert got == status and text in message


@pytest.mark.parametrize("entry,defaults,change", [
    ("miq_rms_fprop", NORM, dict(rows=0, x=None, y=None)),
    ("miq_rms_row8", NORM8, dict(c=0, codes=None)),
    ("miq_rms_bprop", BACK, dict(c=0, dgain=None)),
    ("miq_rms_bprop", BACK, dict(rows=0, accumulate=1, dgain=None, dy=None)),
    ("miq_act_row8", ACT, dict(rows=0, x=None, scales=None)),
    ("miq_row8_expand", EXPAND, dict(rows=0, y=None)),
    ("miq_row8_linear", LINEAR, dict(rows=0, y=None)),
    ("miq_row8_linear", LINEAR, dict(k=0, w_codes=None)),
    ("miq_row8_experts", EXPERTS, dict(rows=0, offsets=None)),
    ("miq_experts_join", JOIN, dict(tokens=0, out=None)),
])
def test_nothing_to_do_enqueues_nothing(entry, defaults, change):
    assert _call(entry, defaults, **change)[0] == _capi.MIQ_OK


def test_workspace_sizes():
    assert M.rms_bprop_workspace_size(0, 64) == 0 == M.rms_bprop_workspace_size(64, 0)
    assert M.rms_bprop_workspace_size(1, 5) == 20
    assert M.rms_bprop_workspace_size(1 << 30, 4096) <= 1280 * 4096 * 4
    assert M.rms_bprop_workspace_size(1 << 17, 1 << 29) == 1 << 31  # one row of it
    assert M.row8_workspace_size(8192, 8192, 2000, 4096) == 0 == M.row8_workspace_size(4, 4, 2001, 4096)
    assert M.row8_workspace_size(8192, 8192, 2001, 4096) == (8192 + 4096) * 2048
    assert M.row8_workspace_size(100, 8192, 2001, 4096, 3) == (100 + 3 * 4096) * 2048
    assert M.row8_workspace_size(0, 8192, 2001, 4096) == 0 == M.row8_workspace_size(10, 0, 2001, 4096)
    with pytest.raises(M.MiqError, match="x_rows"):
        M.row8_workspace_size(-1, 1, 1, 1)
    assert M.lib().miq_row8_workspace_size(1, 1, 1, 1, 1, None) == NULL
    with pytest.raises(M.MiqError, match="2\\^46"):
        M.rms_bprop_workspace_size(1 << 40, 1 << 10)
    assert M.lib().miq_rms_bprop_workspace_size(1, 1, None) == NULL


def test_host_tensors_are_refused():
    x, gain, ids = torch.zeros((3, 8)), torch.zeros(8), torch.zeros((3, 2), dtype=torch.int32)
    kept = M.Row8(x.to(torch.int8), x[:, 0].contiguous())
    w = M.Row8(torch.zeros((2, 4, 8), dtype=torch.int8), torch.zeros((2, 4)))
    for call in (lambda: M.rms_fprop(x, gain), lambda: M.rms_row8(x, gain), lambda: M.rms_bprop(x, x, gain),
                 lambda: M.act_row8(x), lambda: M.row8_expand(kept), lambda: M.row8_linear(kept, kept),
                 lambda: M.row8_experts(kept, w, ids[:, 0].contiguous()), lambda: M.experts_plan(ids, 4),
                 lambda: M.experts_join(x, ids)):
        with pytest.raises(ValueError, match="device memory"):
            call()


@pytest.mark.parametrize("src", ["rms.hip", "rms_grad.hip", "row8.hip", "row8_few.hip", "row8_tile.hip", "experts.hip"])
def test_every_wide_store_is_followed_by_two_wait_states(src, tmp_path):
    dst = tmp_path / "k.s"
    subprocess.run([B.hipcc(), *B.common_flags(), "--cuda-device-only", "-S", str(B.CSRC / src), "-o", str(dst)],
                   check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    short = [g for g in store_gaps(dst.read_text().splitlines()) if g[3] < 2]
    assert not short, short[:5]
