"""Plain references of the paged operators (numpy / torch in 64 bits) and the
tolerances of their tests."""
import numpy as np
import torch

TYPES = {"f32": (torch.float32, torch.float16, 0, 1), "f16": (torch.float16, torch.float16, 1, 1),
         "bf16": (torch.bfloat16, torch.bfloat16, 30, 30)}   # q type, cache type, their ids


def blocks(tokens, page):
    return -(-int(tokens) // page)


def plan(ln, add, release, page, table, free, n_free, rows_cap):
    """t3b_op_kv_plan by its definition; arrays are copied.  None when the step does not fit."""
    ln, add, table, free = [np.array(x, np.int64) for x in (ln, add, table, free)]
    release = np.zeros_like(ln) if release is None else np.array(release, np.int64)
    n, width = table.shape
    if ((ln < 0) | (add < 0) | (release < 0) | (ln + add > width * page) | (release > width * page) |
            ((release > 0) & (ln > 0))).any():
        return None
    stack = list(free[:n_free])
    for i in range(n):
        stack += list(table[i, :blocks(release[i], page)])
    need = sum(blocks(ln[i] + add[i], page) - blocks(ln[i], page) for i in range(n))
    if not 0 <= n_free <= free.size or len(stack) > free.size or need > len(stack) or add.sum() > rows_cap:
        return None
    free[n_free:len(stack)] = stack[n_free:]
    req, pos, slots = ([-1] * rows_cap for _ in range(3))
    starts, r = [0], 0
    for i in range(n):
        for b in range(blocks(ln[i], page), blocks(ln[i] + add[i], page)):
            table[i, b] = stack.pop()
        for t in range(add[i]):
            p = int(ln[i]) + t
            req[r], pos[r], slots[r] = i, p, int(table[i, p // page]) * page + p % page
            r += 1
        starts.append(r)
    return dict(table=table, free=free, n_free=len(stack), row_start=np.array(starts), row_req=np.array(req),
                row_pos=np.array(pos), slots=np.array(slots), len_out=ln + add)


class Batch:
    """A paged cache with prefixes and own keys, random but for the slots that
    no key lies in: those hold NaN, and the table entries past a length hold
    ids outside the pool, so that a read of either shows."""

    def __init__(self, kind, lens, heads, kv_heads, dim, page, prefix_lens=(), prefix_start=None, adds=None, seed=0,
                 gap=0, q_scale=1.0, q_pad=0, spare=3, pages_at=0, device="cuda", share=False):
        g = torch.Generator().manual_seed(seed)
        qt, ct, self.q_id, self.c_id = TYPES[kind]
        self.kind, self.heads, self.kv, self.dim, self.page = kind, heads, kv_heads, dim, page
        self.lens, self.adds = list(lens), None if adds is None else list(adds)
        n, self.prefix_lens = len(lens), list(prefix_lens)
        self.prefix_start = list(prefix_start) if prefix_start is not None else [0] + [n] * len(self.prefix_lens)
        width = max(1, max(blocks(max(x, 0), page) for x in lens)) + 1
        pwidth = max([1] + [blocks(x, page) for x in self.prefix_lens]) + 1
        if share and len(self.prefix_lens) < n:
            # a decode call computes a prefix once for the batch where re-reading it could cost over 48 MB,
            # judged by the room in the prefix table: leave that much room
            pwidth = max(pwidth, blocks(50e6 / (4 * kv_heads * dim * (n - max(1, len(self.prefix_lens)))) + page, page))
        used = sum(blocks(max(x, 0), page) for x in lens) + sum(blocks(x, page) for x in self.prefix_lens)
        self.n_pages = pages_at + used + spare
        ids = (pages_at + torch.randperm(used + spare, generator=g)).tolist()
        far = 1 << 28
        table, ptable = torch.full((n, width), far, dtype=torch.int32), torch.full((max(1, len(self.prefix_lens)), pwidth), far, dtype=torch.int32)
        dense = kv_heads * page * dim
        self.stride = dense + gap
        pool = torch.empty(2, self.n_pages * self.stride, dtype=ct, device=device)
        pool[:, pages_at * self.stride:] = float("nan")
        self.k, self.v = pool[0], pool[1]
        self.own, self.pre = [], []
        view = [x[pages_at * self.stride:].view(-1, self.stride)[:, :dense].view(-1, kv_heads, page, dim) for x in pool]

        def put(count, row):
            kv = torch.randn(2, max(count, 0), kv_heads, dim, generator=g).to(ct)
            for b in range(blocks(max(count, 0), page)):
                row[b] = ids.pop()
                part = kv[:, b * page:(b + 1) * page].to(device)
                for x in range(2):
                    view[x][int(row[b]) - pages_at, :, :part.shape[1]] = part[x].transpose(0, 1)
            return kv

        for i, x in enumerate(lens):
            self.own.append(put(x, table[i]))
        for i, x in enumerate(self.prefix_lens):
            self.pre.append(put(x, ptable[i]))
        self.table, self.ptable = table.to(device), ptable.to(device)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        self.len, self.plen, self.pstart = i32(self.lens), i32(self.prefix_lens or [0]), i32(self.prefix_start)
        self.starts = list(np.cumsum([0] + (self.adds if adds is not None else [1] * n)))
        self.row_start = i32(self.starts)
        self.rows = self.starts[-1]
        w = heads * dim
        self.q_all = (torch.randn(self.rows, w + q_pad, generator=g) * q_scale).to(qt).to(device)
        self.q = self.q_all[:, :w]
        self.out_all = torch.full((self.rows + 2, w + q_pad), -7.0, dtype=qt, device=device)   # two rows behind the last

    def desc(self, pkg, out=None, rows=None, workspace=True):
        out = self.out_all if out is None else out
        prompt = self.adds is not None
        c = pkg.PagedKv(k=self.k.data_ptr(), v=self.v.data_ptr(), page_stride=self.stride, dtype=self.c_id,
                        n_pages=self.n_pages, n_kv_head=self.kv, page_size=self.page, head_dim=self.dim)
        d = pkg.SharedAttn(cache=c, q=self.q.data_ptr(), out=out.data_ptr(), q_stride=self.q_all.stride(0),
                           out_stride=out.stride(0), len=self.len.data_ptr(), table=self.table.data_ptr(),
                           row_start=self.row_start.data_ptr() if prompt else None, dtype=self.q_id, n_head=self.heads,
                           n=len(self.lens), rows=self.rows if rows is None else rows, max_blocks=self.table.shape[1])
        if self.prefix_lens:
            d.prefix_start, d.prefix_len = self.pstart.data_ptr(), self.plen.data_ptr()
            d.prefix_table, d.n_prefix, d.prefix_max_blocks = self.ptable.data_ptr(), len(self.prefix_lens), self.ptable.shape[1]
        if workspace:
            import ctypes
            size = pkg.lib().t3b_op_attention_shared_workspace(ctypes.byref(d))
            self.ws = torch.empty(max(16, size), dtype=torch.uint8, device=self.q.device)
            self.ws.fill_(0xFF)                                  # NaN wherever it is read before it is written
            d.workspace, d.workspace_bytes = self.ws.data_ptr(), size
        return d

    def keys(self, i):
        """K and V of request i in 64 bits, [2][keys][kv heads][dim], prefix first."""
        parts = [self.own[i]]
        for p in range(len(self.prefix_lens)):
            if self.prefix_start[p] <= i < self.prefix_start[p + 1]:
                parts.insert(0, self.pre[p])
        return torch.cat(parts, 1).double()

    def reference(self, scale=None):
        """(out, tolerance) in 64 bits, [rows][heads * dim].

        The tolerance is a bound, worked out per element: with s = scale *
        q.k a score is off by at most ds = (D + 4) 2^-24 * scale * sum |q k|
        (a sum of D products in 32 bits, q split in two parts of 11 bits,
        2^-22) + 2^-22 |s - max| (the exponent's argument), so a weight is off
        by 2 ds (its own and the sum's) + 2^-21 (exp) + keys * 2^-24 (sums in 32
        bits).  16-bit types round each probability too, by eps / 2 of itself
        (f16: at least 2^-25 of the largest); the output is rounded once,
        eps / 2.  All of it multiplies sum w |v|."""
        sc = scale or 1.0 / np.sqrt(self.dim)
        D, g = self.dim, self.heads // self.kv
        out = torch.zeros(self.rows, self.heads, D, dtype=torch.float64)
        tol = torch.zeros_like(out)
        eps = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[self.kind]
        tiny = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}[self.kind]
        half = torch.finfo(self.q.dtype).eps / 2
        q = self.q.cpu().double().reshape(self.rows, self.heads, D)
        for i in range(len(self.lens)):
            kv = self.keys(i)
            rows = slice(self.starts[i], self.starts[i + 1])
            r, L = self.starts[i + 1] - self.starts[i], kv.shape[1]
            if r == 0 or L == 0:
                continue
            K, V = [x.transpose(0, 1).repeat_interleave(g, 0) for x in kv]      # [heads][keys][dim]
            qi = q[rows].transpose(0, 1)
            hide = torch.arange(L)[None] >= (L - r + 1 + torch.arange(r))[:, None]
            if self.adds is None:
                hide[:] = False
            s = (qi @ K.transpose(1, 2)) * sc
            s = s.masked_fill(hide, -np.inf)
            w = s.softmax(-1)
            o = w @ V
            ab = (qi.abs() @ K.abs().transpose(1, 2)) * abs(sc)
            ds = (D + 8) * 2.0 ** -24 * ab + 2.0 ** -22 * (s.amax(-1, keepdim=True) - s).masked_fill(hide, 0.0)
            # a score far below the largest has no weight to be wrong about
            ds = torch.where(w > 1e-12, ds, 0.0).amax(-1, keepdim=True)
            wv = w @ V.abs()
            t = wv * (torch.expm1(2 * ds) + 2.0 ** -21 + L * 2.0 ** -24 + 2 * eps) + half * o.abs() * 1.01 + 2 * L * tiny * V.abs().amax()
            out[rows], tol[rows] = o.transpose(0, 1), t.transpose(0, 1)
        return out.reshape(self.rows, -1), tol.reshape(self.rows, -1) + 1e-30
