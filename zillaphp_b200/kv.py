"""Python handle on the paged K/V cache of libzilla_b200.so (zilla_kv_*)."""
from __future__ import annotations

from ctypes import c_float

from . import native
from .backend import ZillaError

TYPES = {"fp32": 0, "bf16": 1, "fp16": 2}


class PagedKv:
    """K and V of many sequences in pages, [pages][kv_heads][page][head_dim].

    Every tensor argument is a registry handle; integers are int32 in a buffer.  The batch: sequence b's
    new rows are start[b] .. start[b + 1] - 1, len[b] of its own tokens are cached (those included), the
    i-th lies in page pages[b][i // page]; all stand behind the same prefix_len tokens.
    """

    def __init__(self, pages: int, page: int, kv_heads: int, head_dim: int, dtype: str = "bf16"):
        self.lib = native.load()
        self.id = self.lib.zilla_kv_create(pages, page, kv_heads, head_dim, TYPES[dtype])
        if self.id <= 0:
            raise ZillaError(f"zilla_kv_create failed. ({native.last_error()})")
        self.k_id = self.lib.zilla_kv_k_id(self.id)
        self.v_id = self.lib.zilla_kv_v_id(self.id)

    def append(self, x_type: int, q_id: int, q_off: int, q_ld: int, k_id: int, k_off: int, k_ld: int, v_id: int,
               v_off: int, v_ld: int, qout_id: int, start_id: int, len_id: int, pages_id: int, batch: int, rows: int,
               q_heads: int, max_pages: int, prefix_len: int = 0, table_id: int = 0, rot_dim: int = 0,
               interleaved: int = 0) -> None:
        """Stores the new rows' K (rotated) and V in their pages and the rotated Q in qout (zilla_kv_append)."""
        if self.lib.zilla_kv_append(self.id, x_type, q_id, q_off, q_ld, k_id, k_off, k_ld, v_id, v_off, v_ld, qout_id,
                                    start_id, len_id, pages_id, batch, rows, q_heads, max_pages, prefix_len, table_id, rot_dim,
                                    interleaved):
            raise ZillaError(f"zilla_kv_append failed. ({native.last_error()})")

    def attend(self, q_id: int, out_id: int, start_id: int, len_id: int, pages_id: int, prefix_pages_id: int, batch: int,
               rows: int, q_heads: int, max_pages: int, prefix_len: int, max_new: int, max_len: int, scale: float,
               work_id: int = 0) -> None:
        """Attention of the new rows over the prefix and their sequence's own keys (zilla_kv_attend)."""
        if self.lib.zilla_kv_attend(self.id, q_id, out_id, start_id, len_id, pages_id, prefix_pages_id, batch, rows,
                                    q_heads, max_pages, prefix_len, max_new, max_len, c_float(scale), work_id):
            raise ZillaError(f"zilla_kv_attend failed. ({native.last_error()})")

    def attend_work(self, batch: int, rows: int, q_heads: int, prefix_len: int, max_new: int, max_len: int) -> int:
        """Floats of attend's workspace for these sizes (0: none)."""
        n = int(self.lib.zilla_kv_attend_work(self.id, batch, rows, q_heads, prefix_len, max_new, max_len))
        if n < 0:
            raise ZillaError(f"zilla_kv_attend_work failed. ({native.last_error()})")
        return n

    def close(self) -> None:
        if getattr(self, "id", 0) > 0:
            self.lib.zilla_kv_destroy(self.id)
            self.id = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
