"""How tenzo_hip_attn_tree_kv4 shares rows and tokens among workgroups (kv4_plan in
csrc/attention_kv4.hip, for trees), stated once more, so that a test can say which kernel it means
to run. test_tree_refusals.py holds it against the workspaces that the library asks for."""
from tests import kv4_plan
from tests.kv4_plan import PAGE, RECORD, TILE, _up


def plan(T, B, Hq, Hkv, width, cu, half):
    """(kernel, splits, bytes of workspace), as kv4_plan.plan has them."""
    G, ctx = Hq // Hkv, width * PAGE
    per = _up(T * G, B) if cu else G
    tiles = T * Hq / 128
    if per > 44 and (ctx <= 1024 and tiles > (110 if half else 360) or
                     ctx <= 2048 and tiles > (360 if half else 600)):
        return "128", 1, 0
    if per > (40 if half else 56) and ctx > 1024 and T * Hq * ctx > (14e6 if half else 22e6):
        most = (T * G // 128 + B) * Hkv * (_up(ctx, TILE) + 4)
        return "128 even", 1, min(_up(most, 4), 512) * 2 * 128 * RECORD
    # (the prompts' kernel serves no trees)
    name, splits, size = kv4_plan.plan(T, B, Hq, Hkv, width, cu)
    return (name, splits, size) if name != "128" else _sixteen(T, B, G, Hkv, ctx, cu, per)


def _sixteen(T, B, G, Hkv, ctx, cu, per):
    """What kv4_plan.plan gives where it does not choose the prompts' kernel."""
    rows = 4 if per <= 4 else 16
    rt = 32 if per > 16 and T * G // 16 * Hkv > 512 and ctx <= 1024 else rows
    units = T * G // rt + B if cu else B * _up(G, rt)
    step = 128 if rt == 32 else 256
    steps = _up(ctx, step) if ctx else 1
    room, most = 512 if rows == 16 else 768, units * Hkv * (steps + 1)
    if rt == rows and B > 1 and units * Hkv < 2 * room < 2 * units * Hkv * steps:
        return f"{rows} even", 1, min(most, room) * 2 * rows * RECORD
    likely = max(_up(T * G, rt), B) if cu else units
    own, fits = T / B / ctx if ctx else 0.0, room / (likely * Hkv)
    s = 1 + int((fits - 1) / (1 - 0.5 * min(own, 1.0))) if fits > 1 else 1
    chunk = _up(steps, min(s, steps)) * step
    splits = _up(ctx, chunk) if ctx else 1
    return str(rt), splits, T * G * Hkv * splits * RECORD if splits > 1 else 0
