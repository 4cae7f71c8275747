"""The paged cache's operators in plain torch, on any device.  TEST INFRASTRUCTURE: it lets the engine's paged schedules run on the CPU, and gives a
whole model on the GPU something to be compared with."""
import torch

E4M3 = torch.float8_e4m3fn


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


class PagedOps:
    @staticmethod
    def rope_paged_store(qkv, table, input_pos, sequence, pages, q_out, k_pages, v_pages, k_scale, v_scale, n_head, halves, tokens, pages_shape,
                         cache_shape):
        n_pages, n_kv, page, dim = cache_shape
        pos = input_pos.long()
        seq = torch.arange(tokens, device=qkv.device) if sequence is None else sequence.long()
        live = (pos >= 0) & (pos < pages_shape[1] * page) & (seq >= 0) & (seq < pages_shape[0])
        if table is not None:
            live &= pos < table.shape[0]
        ids = pages[seq.clamp(0, pages_shape[0] - 1), (pos // page).clamp(0, pages_shape[1] - 1)].long()
        live &= (ids >= 0) & (ids < n_pages)
        x = qkv[live].float().view(-1, n_head + 2 * n_kv, dim)
        if table is not None:
            c, s = table[pos[live]].float().unsqueeze(1).unbind(-1)
            half = table.shape[1]
            a, b = (slice(0, half), slice(half, 2 * half)) if halves else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
            x0, x1 = x[:, :n_head + n_kv, a].clone(), x[:, :n_head + n_kv, b].clone()
            x[:, :n_head + n_kv, a], x[:, :n_head + n_kv, b] = x0 * c - x1 * s, x1 * c + x0 * s
        q_out[live] = x[:, :n_head].to(q_out.dtype)
        at = ids[live], pos[live] % page
        for new, stored, scales in ((x[:, n_head:n_head + n_kv], k_pages, k_scale), (x[:, n_head + n_kv:], v_pages, v_scale)):
            if scales is not None:
                top = new.abs().amax(-1).clamp(min=2.0 ** -100)
                scales[at[0], :, at[1]] = top / 448
                new = (new * 448 / top.unsqueeze(-1)).clamp(-448, 448)
            _bytes(stored)[at[0], :, at[1]] = _bytes(new.to(stored.dtype))

    @staticmethod
    def paged_attn_workspace_bytes(n_head, n_kv, head_dim):
        return 0

    @staticmethod
    def _rows(stored, scales, pages, b, lo, hi):
        page = stored.shape[2]
        at = torch.arange(lo, hi, device=pages.device)
        ids = pages[b].long()[at // page]
        at, ids = at[ids >= 0], ids[ids >= 0]
        x = _bytes(stored)[ids, :, at % page].view(stored.dtype).float()
        return x if scales is None else x * scales[ids, :, at % page].unsqueeze(-1)

    @classmethod
    def paged_attention(cls, q, k_pages, v_pages, k_scale, v_scale, pages, input_pos, window, scale, out, workspace, n_head, pages_shape, cache_shape):
        for b, pos in enumerate(input_pos.tolist()):
            lo = max(0, pos + 1 - window) if window else 0
            k, v = (cls._rows(t, s, pages, b, lo, max(pos + 1, 0)).transpose(0, 1) for t, s in ((k_pages, k_scale), (v_pages, v_scale)))
            w = torch.softmax(q[b].float().view(k.shape[0], -1, k.shape[2]) @ k.transpose(1, 2) * scale, -1)
            out[b] = (w @ v).reshape(out[b].shape).to(out.dtype)

    @classmethod
    def paged_load(cls, k_pages, v_pages, k_scale, v_scale, pages, last_pos, k_out, v_out, rows, pages_shape, cache_shape):
        for b, last in enumerate(last_pos.tolist()):
            n = min(last + 1, rows)
            for t, s, out in ((k_pages, k_scale, k_out), (v_pages, v_scale, v_out)):
                out[b, :, :n] = cls._rows(t, s, pages, b, 0, n).transpose(0, 1).to(out.dtype)
                out[b, :, n:-(-n // 64) * 64] = 0
