"""Forward-mode derivatives of the gated delta rule's entry points: refused, on any machine, since
the kernels would drop a dual tensor's tangent."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad

import omegalax_amd as om
from omegalax_amd.deltanet import recurrent_gated_delta_rule_step

BF = torch.bfloat16
CFG = dict(num_k_heads=1, head_k_dim=64, num_v_heads=2, head_v_dim=64)


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


QKV = [z(1, 4, 1, 64), z(1, 4, 1, 64), z(1, 4, 2, 64), z(1, 4, 2), z(1, 4, 2)]
STATE = z(1, 2, 64, 64, dtype=torch.float32)
MIXED = [z(1, 4, 256), z(1, 4, 2, 64), z(1, 4, 2), z(1, 4, 2), z(256, 4), z(2), z(2), z(64)]
CALLS = {
    "chunk": (lambda *x: om.chunk_gated_delta_rule(*x[:5], initial_state=x[5]), QKV + [STATE]),
    "chunk_bwd": (lambda *x: om.chunk_gated_delta_rule_bwd(*x[:6], initial_state=x[6], d_final_state=x[7]),
                  QKV + [z(1, 4, 2, 64), STATE, STATE]),
    "recurrent": (recurrent_gated_delta_rule_step, [t[:, 0] for t in QKV] + [STATE]),
    "prefill": (lambda *x: om.gdn_prefill(*x[:8], initial_state=x[8], conv_state=x[9], **CFG),
                MIXED + [STATE, z(1, 256, 3)]),
    "prefill_bwd": (lambda *x: om.gdn_prefill_bwd(*x[:9], initial_state=x[9], d_final_state=x[10], **CFG),
                    MIXED + [z(1, 4, 128), STATE, STATE]),
    "decode": (lambda *x: om.gdn_decode_step(*x, **CFG),
               [t[:, 0] for t in MIXED[:4]] + MIXED[4:] + [z(1, 256, 3), STATE]),
    "ab": (om.gdn_ab_projections, [z(4, 64), z(2, 64), z(2, 64)]),
    "qkv_conv": (om.qkv_conv_projection, [z(4, 64), z(256, 64), z(256, 4)]),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_dual_tensor_is_refused(name):
    call, args = CALLS[name]
    with forward_ad.dual_level():
        for i in range(len(args)):
            x = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*x)
        with pytest.raises(ValueError, match="GPU"):  # a level alone changes nothing
            call(*args)
