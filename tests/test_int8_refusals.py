"""What the C entry points of the 8-bit integer products and of the balance
loss refuse, and what they take without a launch: no GPU is needed, since
every check comes before the first launch."""
import ctypes as C

from chimere_amd import _lib

P = C.c_void_p(0x1000)      # 4096: aligned, never read
ODD = C.c_void_p(0x1008)
MORE = 1 << 40


def err():
    L = _lib.lib()
    msg = L.chimere_hip_get_last_error_string().decode()
    return L.chimere_hip_get_last_error(), msg


def refuses(name, good, **changes):
    """The call with each change of one argument (position: value) is refused with its code."""
    for what, (at, value, code) in changes.items():
        args = list(good)
        args[at] = value
        getattr(_lib.lib(), name)(*args)
        got, msg = err()
        assert got == code and name[len("chimere_"):].split("_loss")[0] in msg, (name, what, got, msg)


def test_quantize():
    good = [0, P, 64, P, 64, P, 4, 64, None]
    refuses("chimere_quantize_i8", good, type=(0, 2, 1), x=(1, None, 1), q=(3, None, 1), scale=(5, None, 1), rows=(6, -1, 1),
            cols=(7, 0, 1), x_stride=(2, -1, 1), q_short=(4, 48, 1), q_stride=(4, 72, 1), q_ptr=(3, ODD, 1),
            too_many=(6, 1 << 31, 1), x_align=(1, C.c_void_p(0x1002), 1))
    good[6] = 0
    _lib.lib().chimere_quantize_i8(*good)           # no rows: nothing to do
    assert err()[0] == 0


def test_gemm():
    good = [P, 64, P, P, 64, P, None, 0, P, 32, 4, 32, 64, None]
    refuses("chimere_gemm_i8", good, a=(0, None, 1), lda=(1, 48, 1), lda_align=(1, 72, 1), a_align=(0, ODD, 1), a_scale=(2, None, 1),
            w=(3, None, 1), w_align=(3, ODD, 1), ldw=(4, 63, 1), ldw_far=(4, 1 << 24, 1), w_scale=(5, None, 1), type=(7, 8, 1),
            out=(8, None, 1), ldo=(9, 31, 1), ntok=(10, -1, 1), nrows=(11, 0, 1), ncols=(12, 0, 1), long=(12, 131072, 1),
            out_align=(8, C.c_void_p(0x1002), 1), many_tok=(10, (1 << 25) + 1, 1), many_rows=(11, 0x7FFFFFFF, 1))
    good[10] = 0
    _lib.lib().chimere_gemm_i8(*good)
    assert err()[0] == 0


def test_linear():
    L = _lib.lib()
    need = L.chimere_linear_i8_workspace_size(4, 100)
    assert need >= 4 * 112 + 16
    assert L.chimere_linear_i8_workspace_size(0, 100) == 0 == L.chimere_linear_i8_workspace_size(4, 131072)
    good = [1, P, 100, P, 112, P, None, 30, P, 32, 4, 32, 100, P, need, None]
    refuses("chimere_linear_i8", good, type=(0, 13, 1), x=(1, None, 1), x_stride=(2, -4, 1), w=(3, None, 1), ldw=(4, 100, 1),
            out_type=(7, 2, 1), out=(8, None, 1), ldo=(9, 31, 1), ncols=(12, 1 << 20, 1), ws=(13, None, 1), ws_align=(13, ODD, 3),
            ws_small=(14, need - 1, 3))


def test_moe():
    L = _lib.lib()

    def layer(**kw):
        c = _lib.MoeI8LayerC(256, 128, 8, *[0x1000] * 6)
        for k, v in kw.items():
            setattr(c, k, v)
        return C.byref(c)

    need = L.chimere_moe_i8_workspace_size(layer(), 2, 4)
    assert 0 < need <= L.chimere_moe_i8_workspace_size(layer(), 2, 100)
    assert L.chimere_moe_i8_workspace_size(layer(), 17, 4) == 0 == L.chimere_moe_i8_workspace_size(layer(hidden=250), 2, 4)
    assert L.chimere_moe_i8_workspace_size(None, 2, 4) == 0 == L.chimere_moe_i8_workspace_size(layer(), 2, 0)
    good = [layer(), 0, P, 256, P, P, 2, 30, P, 256, 4, P, need, None]
    refuses("chimere_moe_i8", good, layer=(0, None, 1), type=(1, 8, 1), x=(2, None, 1), ids=(4, None, 1), wts=(5, None, 1),
            k=(6, 17, 1), k0=(6, 0, 1), out_type=(7, 12, 1), out=(8, None, 1), ldo=(9, 255, 1), ntok=(10, -1, 1),
            far=(10, (1 << 31) // 256, 1), ws=(11, None, 1), ws_align=(11, ODD, 3), ws_small=(12, need - 1, 3),
            hidden=(0, layer(hidden=248), 1), ffn=(0, layer(ffn=0), 1), many=(0, layer(n_experts=1025), 1),
            gate=(0, layer(gate=None), 1), align=(0, layer(down=0x1008), 1), scale=(0, layer(up_scale=None), 1))
    good[10] = 0
    L.chimere_moe_i8(*good)
    assert err()[0] == 0


def test_balance():
    L = _lib.lib()
    need = L.chimere_balance_loss_workspace_size(256, 1000)
    assert need > 0 == L.chimere_balance_loss_workspace_size(1025, 10)
    good = [0, P, 256, P, 8, None, P, P, P, P, 256, 1000, P, need, None]
    refuses("chimere_balance_loss", good, type=(0, 8, 1), logits=(1, None, 1), stride=(2, -1, 1), ids=(3, None, 1), k=(4, 0, 1),
            loss=(6, None, 1), probs=(7, None, 1), counts=(8, None, 1), tokens=(9, None, 1), many=(10, 1025, 1), none=(10, 0, 1), far=(11, 1 << 30, 1), wide=(4, 1025, 1),
            ntok=(11, -1, 1), ws=(12, None, 1), ws_align=(12, ODD, 3), ws_small=(13, need - 1, 3))
    good = [0, P, 256, None, P, P, P, 8, P, 256, 256, 1000, None]
    refuses("chimere_balance_loss_grad", good, align=(1, C.c_void_p(0x1002), 1), grad_align=(8, C.c_void_p(0x1001), 1), type=(0, 2, 1), logits=(1, None, 1), counts=(4, None, 1), tokens=(5, None, 1),
            grad_loss=(6, None, 1), k=(7, 0, 1), grad=(8, None, 1), ldg=(9, 255, 1), many=(10, 2000, 1), ntok=(11, -1, 1))
    good[11] = 0
    L.chimere_balance_loss_grad(*good)
    assert err()[0] == 0
