"""Operands that share memory with what a call writes are refused by their addresses alone (no GPU)."""
import axon_b200 as ax

AT = 1 << 20  # addresses that nothing looks behind


def _refused(status):
    """Whether a call was refused for an overlap; without a GPU every other one ends at its first pointer."""
    return status == ax.Status.ERR_INVALID and b"must not overlap" in ax.lib().axq_last_error()


def test_quantize_f8_padding():
    """The bytes between cols and ld in the last block of 128 columns are set to 0, those of the last row too."""
    L = ax.lib()

    def call(codes, scales, src=AT, rows=1, cols=4, ld=16, block_rows=1):
        return _refused(L.axq_quantize_f8(0, src, codes, ld, scales, rows, cols, block_rows, None))

    c = 2 * AT
    assert call(c, c + 4) and call(c, c + 12) and not call(c, c + 16)
    assert call(c, c + 32 + 8, rows=3) and not call(c, c + 48, rows=3)
    # a row stride beyond the block: what lies behind it is left as it is
    assert call(c, c + 124, ld=256) and not call(c, c + 128, ld=256)
    assert call(c, c + 256 + 124, rows=2, ld=256, block_rows=128)
    assert call(c, 3 * AT, src=c + 8) and not call(c, 3 * AT, src=c + 16) and call(c, 3 * AT, src=3 * AT)


def test_linear_f8():
    """Neither y nor the workspace may share memory with an operand or with the other."""
    L = ax.lib()
    names = ("w", "ws", "x", "xs", "bias", "y", "work")
    M, K, N = 256, 256, 4

    def call(x_type, **at):
        p = {n: (i + 1) * 16 * AT for i, n in enumerate(names)}
        p.update(at)
        packed = x_type == 3
        return _refused(L.axq_linear_f8(p["w"], K, p["ws"], x_type, p["x"], K, p["xs"] if packed else None, p["bias"], 0, p["y"],
                                        M, K, N, p["work"], 1 << 20, None))

    at = {n: (i + 1) * 16 * AT for i, n in enumerate(names)}
    size = {"w": M * K, "ws": 4 * 4, "xs": N * 2 * 4, "bias": 4 * M}
    for x_type, x_size in ((0, 4 * N * K), (2, 2 * N * K), (3, N * K)):
        assert not call(x_type)
        work = L.axq_linear_f8_workspace_size(x_type, K, N)
        for n, nbytes in {**size, "x": x_size, "work": work}.items():
            if n == "xs" and x_type != 3:
                continue
            assert call(x_type, y=at[n] + nbytes - 4) and call(x_type, y=at[n] - 4 * N * M + 4), (x_type, n)
            assert not call(x_type, y=at[n] + nbytes) and not call(x_type, y=at[n] - 4 * N * M), (x_type, n)
            if n != "work":
                assert call(x_type, work=at[n] + nbytes - 1) and call(x_type, work=at[n] - work + 1), (x_type, n)
                assert not call(x_type, work=at[n] + nbytes) and not call(x_type, work=at[n] - work), (x_type, n)
    # operands that are only read may be the same memory
    assert not call(3, x=at["w"], xs=at["ws"], bias=at["ws"])


def test_moe_route():
    L = ax.lib()
    T, E, K, H = 5, 8, 2, 96
    at = {n: (i + 1) * AT for i, n in enumerate(("x", "router", "ids", "p"))}

    def call(dtype=0, **kw):
        p = {**at, **kw}
        return _refused(L.axq_moe_route(dtype, p["x"], p["router"], p["ids"], p["p"], T, E, K, H, 1, None))

    out = 4 * T * K
    assert not call()
    for dtype, size in ((0, 4), (1, 2)):
        for n, nbytes in (("x", size * T * H), ("router", 4 * E * H)):
            for o in ("ids", "p"):
                assert call(dtype, **{o: at[n] + nbytes - 4}) and call(dtype, **{o: at[n] - out + 4})
                assert not call(dtype, **{o: at[n] + nbytes}) and not call(dtype, **{o: at[n] - out})
    assert call(ids=at["p"] + out - 4) and not call(ids=at["p"] + out)
    assert not call(x=at["router"])


def _apart(call, at, sizes, written):
    """Every range in `written` against every other: refused at the last and the first shared byte, else not."""
    assert not call()
    for o in written:
        for n, nbytes in sizes.items():
            if n != o:
                assert call(**{o: at[n] + nbytes - 4}) and call(**{o: at[n] - sizes[o] + 4}), (o, n)
                assert not call(**{o: at[n] + nbytes}) and not call(**{o: at[n] - sizes[o]}), (o, n)


def test_moe_layer():
    L = ax.lib()
    T, E, K, H, F = 5, 8, 2, 256, 128
    for fmt, gate, down in ((5, E * F * 144, E * H * 144), (64, E * F * H, E * H * F)):
        f8 = fmt == 64
        sizes = {"gate": gate, "up": gate, "down": down, "x": 4 * T * H, "router": 4 * E * H, "ids": 4 * T * K, "p": 4 * T * K,
                 "y": 4 * T * H, "work": L.axq_moe_workspace_size(T, K, H, F)}
        if f8:
            sizes.update({n + "_s": 4 * E * (F // 128) * (H // 128) for n in ("gate", "up", "down")})
        at = {n: (i + 1) * 64 * AT for i, n in enumerate(sizes)}

        def weights(p):
            return [v for n in ("gate", "up", "down") for v in ([fmt] if n != "up" else []) + [p[n], p.get(n + "_s")]]

        def layer(**kw):
            p = {**at, **kw}
            return _refused(L.axq_moe(*weights(p), 0, p["x"], p["router"], 1, p["ids"], p["p"], p["y"], T, E, K, H, F, p["work"],
                                      1 << 40, None))

        def mlp(**kw):
            p = {**at, **kw}
            return _refused(L.axq_moe_mlp(*weights(p), 0, p["x"], p["ids"], p["p"], p["y"], T, E, K, H, F, p["work"], 1 << 40,
                                          None))

        _apart(layer, at, sizes, ("y", "work", "ids", "p"))
        del sizes["router"]
        _apart(mlp, at, sizes, ("y", "work"))
        assert not mlp(up=at["gate"]) and not mlp(ids=at["x"])  # only read
