"""How tenzo_hip_attn_kv4 shares rows and tokens among workgroups (kv4_plan in
csrc/attention_kv4.hip), stated once more, so that a test can say which kernel it means to run.
test_kv4_plan.py holds it against the workspaces that the library asks for."""
PAGE, TILE, RECORD = 16, 64, 128 * 4 + 8


def _up(a, b):
    return -(-a // b)


def plan(T, B, Hq, Hkv, width, cu):
    """(kernel, splits, bytes of workspace); kernel: "4", "16", "32" or "128" rows a workgroup,
    with " even" behind it where the steps are dealt evenly."""
    G, ctx = Hq // Hkv, width * PAGE
    per = _up(T * G, B) if cu else G
    rows = 4 if per <= 4 else 16
    units128 = T * G * Hkv / 128
    rw = 1
    if per > 64 and (units128 > 320 or units128 * ctx > 3500 * TILE):
        rw = 8
    elif per > 16 and T * G // 16 * Hkv > 512 and ctx <= 1024:
        rw = 2
    rt = rows * rw
    units = T * G // rt + B if cu else B * _up(G, rt)
    step = TILE if rw > 4 else TILE * (4 // rw)
    steps = _up(ctx, step) if ctx else 1
    room = 512 if rows == 16 else 768
    most = units * Hkv * (steps + 1)
    if rw == 1 and B > 1 and units * Hkv < 2 * room and units * Hkv * steps > room \
            and most < 2 ** 31:
        return f"{rows} even", 1, min(most, room) * 2 * rows * RECORD
    likely = max(_up(T * G, rt), B) if cu else units
    own = T / B / ctx if ctx else 0.0
    fits = room / (likely * Hkv)
    s = 1 + int((fits - 1) / (1 - 0.5 * min(own, 1.0))) if fits > 1 else 1
    chunk = _up(steps, min(s, steps)) * step
    splits = _up(ctx, chunk) if ctx else 1
    return str(rt), splits, T * G * Hkv * splits * RECORD if splits > 1 else 0
