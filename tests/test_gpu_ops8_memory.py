"""What the workspace of the gated block's gradients from a checkpoint holds, as dp_amd.h states it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,d,f,o", [(64, 64, 512, 4096), (64, 2048, 2048, 2048), (512, 128, 256, 8192), (192, 1600, 240, 8),
                                     (2048, 256, 512, 256), (512, 2048, 512, 1), (4096, 128, 512, 1)])
def test_workspace(dp, n, d, f, o):
    """Restored x, dg, du and h, dh in each of its slices (or g and u, or nothing in their place with up to four
    outputs), and beside them the largest product's slices. Sizes of whole chunks: nothing is copied."""
    ops, b = dp.ops.Operators(), 2
    shape = dp.ops.GatedShape(n, d, f, o, dtype="bf16")
    kept = torch.zeros(dp.ops.keep8_bytes(n, d), dtype=torch.uint8, device="cuda")
    arrays = {k: torch.zeros(s, dtype=torch.bfloat16, device="cuda") for k, s in
              (("wg", (d, f)), ("wu", (d, f)), ("wd", (f, o)), ("dy", (n, o)), ("dx", (n, d)), ("dwg", (d, f)),
               ("dwu", (d, f)), ("dwd", (f, o)))}
    ops.gated_backward8(shape, kept.data_ptr(), *(t.data_ptr() for t in arrays.values()))
    torch.cuda.synchronize()
    plan = shape.plan8()
    few = o <= 4
    held = b * n * (d + (2 if few else 3) * f)
    held += 4 * n * f * plan["dh"][2] if not few else 8 * n * f if "gate" in plan else 0
    outs = {"gate": 2 * n * f, "gate_back": 2 * n * f, "dx": n * d, "dw": 2 * d * f, "dw_down": f * o}
    slices = [4 * outs[k] * plan[k][2] for k in outs if k in plan and plan[k][2] > 1]
    # (up to four outputs: sums of h dy over 16 rows or more, or over 64 slices or fewer of the rows)
    slices.append(4 * f * o * max(64, n // 16) if few else 0)
    used = ops.device_bytes()
    # (an eighth more than asked for, and regions of whole 256 bytes)
    assert held < used <= (held + max(slices) + 20 * 256) * 1.125, (used, held, slices, plan)
