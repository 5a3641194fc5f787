"""Which kernel takes an attention call over the 8-bit cache, by the rule of
csrc/attend8.hip restated: tests name the kernel that each of their cases is for,
so that a change of the rule cannot leave one untested without a failure here."""
import ctypes

import torch

CUS = 256                 # MI355X, and what the library assumes without a GPU
WHOLE, SPLIT, TILE, TILES = "row kernel, one launch", "row kernel, split", "tile kernel, one part", "tile kernel, parts"


def _plan(B, Hq, H, T, D, G, W, max_tokens):
    rows, pairs, cap = Hq // H * T, B * H, W * G
    tokens = min(max_tokens, cap) if max_tokens else cap
    DP = 64 if D <= 64 else 128 if D <= 128 else 256
    whole = DP <= 128 and tokens * DP <= 1024 * 128 and (pairs <= 4096 if rows <= 32 else pairs * -(-rows // 32) <= CUS)
    if whole:
        return WHOLE, 0
    up = lambda n: -(-n // 16) * 16  # noqa: E731
    if rows > (32 if DP == 256 else 64):
        items = pairs * -(-rows // 128)
        parts = max(1, min((1 if DP == 256 else 2) * CUS // items, tokens // 256))
        slots = items * parts if parts > 1 else 0
        return (TILES if parts > 1 else TILE), up(slots * 128 * DP * 4) + up(slots * 128 * 8)
    blocks = 1 if rows <= 16 else 2 if rows <= 32 or DP == 256 else 3 if rows <= 48 else 4
    items = pairs * -(-rows // (16 * blocks))
    groups = (2 if DP <= 128 and DP * blocks <= 256 else 1) * CUS
    slots = 2 * min(groups, items * (2 + -(-cap // 128)))
    return SPLIT, up(slots * 16 * blocks * DP * 4) + up(slots * 16 * blocks * 8) + up(items * 8)


def plan(B, Hq, H, T, D, G, W, max_tokens=0):
    """The kernel's name; what the library asks as workspace has to be that plan's."""
    from kitty import _hip
    name, size = _plan(B, Hq, H, T, D, G, W, max_tokens)
    c = _hip.Cache8(4096, 8192, 16384, H * G * D, G * D, D, H * G * D, G * D, D, 2 * H, 2, 4, H, D, G)
    a = _hip.Cache8AttentionArgs()
    a.batch, a.num_q_heads, a.tokens, a.table_pages, a.plan_tokens, a.sm_scale = B, Hq, T, W, max_tokens, 1.0
    got = ctypes.c_size_t(0)
    L = _hip.load()
    assert L.kitty_cache8_attention_workspace_size(ctypes.byref(c), ctypes.byref(a), ctypes.byref(got)) == _hip.KITTY_OK
    assert got.value == size, (name, size, got.value)
    return name


def planned(cache, q, table, max_tokens=0):
    B, Hq, T, D = q.shape
    return plan(B, Hq, cache.num_kv_heads, T, D, cache.page_tokens, table.shape[1], max_tokens)


def widened(table, cols, value=1 << 30):
    """The table with columns that name no pages: lengths on the device decide, not the table's width."""
    pad = torch.full((table.shape[0], max(0, cols - table.shape[1])), value, dtype=torch.int32, device=table.device)
    return torch.cat([table, pad], 1)
