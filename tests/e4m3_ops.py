"""The operators of projections in 8 bits in plain torch, on any device.  TEST INFRASTRUCTURE: it lets the engine's schedules run on the CPU, and gives a
whole model on the GPU something to be compared with."""
import torch

from e4m3_util import activation64, quantised
from gpt_fast import _C

ACTIVATION = {number: name for name, number in _C.ACTIVATIONS.items()}


def _store(rows, x):
    codes, scale = rows
    got, s = quantised(x)
    codes[:x.shape[0], :x.shape[1]].view(torch.uint8).copy_(got.view(torch.uint8))
    scale[:x.shape[0]] = s


def _values(rows, n):
    codes, scale = rows
    return codes[:n].float() * scale[:n].unsqueeze(1)


class E4M3Ops:
    @staticmethod
    def quantize_rows_e4m3(x, codes, scale, rows, cols, x_ld, codes_ld, early=False):
        _store((codes, scale), x[:rows])

    @staticmethod
    def add_rmsnorm_e4m3(residual, add1, add2, weight, eps, residual_out, codes, scale, rows, dim, codes_ld, residual_scale=1.0, early=False):
        x = residual[:rows] if residual_scale == 1.0 else residual[:rows] * residual_scale
        for add in (add1, add2):
            x = x if add is None else x + add[:rows]
        x = x.clone()
        if residual_out is not None:
            residual_out[:rows] = x
        _store((codes, scale), x.float() * weight.float())
        scale[:rows] *= torch.rsqrt(x.float().square().mean(-1) + eps)

    @staticmethod
    def linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias=None, addend=None, activation=0, glu=(0.0, 0.0, 0.0)):
        z = _values(x, rows) @ _values(w, None).t()
        if activation == _C.ACT_GLU:
            alpha, limit, offset = glu
            up, gate = z.chunk(2, -1)
            gate = gate.clamp(max=limit)
            y = gate * torch.sigmoid(alpha * gate) * (up.clamp(-limit, limit) + offset)
        else:
            y = activation64(ACTIVATION[activation], z if bias is None else z + bias.float())
            if addend is not None:
                y = y + addend.view(-1, n)[:rows].float()
        out.view(-1, n)[:rows] = y.to(out.dtype)

    @staticmethod
    def rope_kvcache(qkv, table, table_gathered, input_pos, q_out, k_cache, v_cache, B, S, n_head, n_kv, head_dim):
        from oracle import ladder_oracle as lo
        rows, pos = B * S, input_pos.long()
        q, k, v = qkv[:rows].view(B, S, -1).split([n_head * head_dim, n_kv * head_dim, n_kv * head_dim], dim=-1)
        turn = table[:S] if table_gathered else table[pos]
        k_cache[:B, :, pos] = lo.rope(k.reshape(B, S, n_kv, head_dim), turn).transpose(1, 2)
        v_cache[:B, :, pos] = v.reshape(B, S, n_kv, head_dim).transpose(1, 2)
        q_out[:rows] = lo.rope(q.reshape(B, S, n_head, head_dim), turn).reshape(rows, n_head * head_dim)


def to_8_bits_and_back(x):
    codes, scale = quantised(x)
    return (codes.float() * scale.unsqueeze(-1)).to(torch.bfloat16)


def faked_ops(vocab):
    """Operators of 16 bits whose projections' inputs go to 8 bits and back (the output projection's, of `vocab` rows, do not)."""
    from cpu_ops import CpuOps

    class Faked(CpuOps):
        @staticmethod
        def linear(x, w, out, rows, addend=None, workspace=None):
            CpuOps.linear(x if w.shape[0] == vocab else to_8_bits_and_back(x[:rows]), w, out, rows, addend, workspace)

        @staticmethod
        def qkv_rope_kvcache(x, *args):
            CpuOps.qkv_rope_kvcache(to_8_bits_and_back(x), *args)

        @staticmethod
        def gateup_swiglu(x, w1, h, rows, workspace):
            CpuOps.gateup_swiglu(to_8_bits_and_back(x[:rows]), w1, h, rows, workspace)
    return Faked


def fake_weights(model):
    """The layers' weights to 8 bits and back."""
    for m in model.layers.modules():
        if isinstance(m, torch.nn.Linear):
            m.weight.data = to_8_bits_and_back(m.weight.data)
