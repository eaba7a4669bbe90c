"""Block-manager factory for the paged KV cache.

The native implementation lives in ``csrc/runtime/block_manager.cpp`` (module
``axrl_b200._runtime``).  When the module has not been built yet (fresh
checkout on a CPU-only machine) it is built on first use with g++; the pure
Python :class:`PyBlockManager` (same semantics, used to cross-check the native
one in tests) is the last resort.
"""

from __future__ import annotations

from collections import OrderedDict

from axrl_b200.ops import _ext


def runtime_module():  # noqa: ANN201
    try:
        return _ext.load("_runtime")
    except Exception:  # noqa: BLE001
        from axrl_b200.csrc.build import build

        build(only="_runtime")
        return _ext.load("_runtime")


def make_block_manager(num_pages: int, page_size: int, prefer_native: bool = True):  # noqa: ANN201
    if prefer_native:
        try:
            return runtime_module().BlockManager(num_pages, page_size)
        except Exception:  # noqa: BLE001
            pass
    return PyBlockManager(num_pages, page_size)


def _mix64(h: int, v: int) -> int:
    M = (1 << 64) - 1
    z = (h ^ ((v + 0x9E3779B97F4A7C15 + ((h << 6) & M) + (h >> 2)) & M)) & M
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
    return z ^ (z >> 31)


class _Node:
    """Content of a cached page: its tokens behind those of ``parent``; outlives its page (``page < 0``) as long as nodes hang on it."""

    __slots__ = ("parent", "hash", "tokens", "page", "children")

    def __init__(self, parent: _Node | None, h: int, tokens: list[int]) -> None:
        self.parent, self.hash, self.tokens, self.page, self.children = parent, h, tokens, -1, 0

    def holds(self, parent: _Node | None, tokens: list[int]) -> bool:
        return self.parent is parent and self.tokens == list(tokens)


class PyBlockManager:
    """Pure-Python twin of the native BlockManager (identical hashing and eviction order)."""

    def __init__(self, num_pages: int, page_size: int) -> None:
        self.page_size, self.num_pages = page_size, num_pages
        self.ref = [0] * num_pages
        self.free = list(range(num_pages - 1, -1, -1))
        self.lru: OrderedDict[int, None] = OrderedDict()
        self.nodes: dict[int, _Node] = {}
        self.node_of: list[_Node | None] = [None] * num_pages

    def num_available(self) -> int:
        return len(self.free) + len(self.lru)

    def num_free(self) -> int:
        return len(self.free)

    def num_cached(self) -> int:
        return sum(n is not None for n in self.node_of)

    def allocate(self, n: int) -> list[int]:
        if n > self.num_available():
            raise RuntimeError("KV cache out of pages")
        out = []
        for _ in range(n):
            if not self.free:
                p, _ = self.lru.popitem(last=False)
                node, self.node_of[p] = self.node_of[p], None
                node.page = -1
                self._trim(node)
                self.free.append(p)
            p = self.free.pop()
            self.ref[p] = 1
            out.append(p)
        return out

    def incref(self, pages: list[int]) -> None:
        for p in pages:
            if self.ref[p] == 0 and self.node_of[p]:
                del self.lru[p]
            self.ref[p] += 1

    def release(self, pages: list[int]) -> None:
        for p in pages:
            if self.ref[p] <= 0:
                raise RuntimeError("double free of KV page")
            self.ref[p] -= 1
            if self.ref[p] == 0:
                if self.node_of[p]:
                    self.lru[p] = None
                else:
                    self.free.append(p)

    def _page_hash(self, h: int, t: list[int], i: int) -> int:
        for j in range(i * self.page_size, (i + 1) * self.page_size):
            h = _mix64(h, t[j] & ((1 << 64) - 1))
        return _mix64(h, 0xC0FFEE + i)

    def _trim(self, n: _Node | None) -> None:
        while n is not None and n.page < 0 and n.children == 0:
            del self.nodes[n.hash]
            n = n.parent
            if n is not None:
                n.children -= 1

    def match_prefix(self, tokens: list[int]) -> tuple[list[int], int]:
        P, pages, h, at = self.page_size, [], 0, None
        for i in range(len(tokens) // P):
            h = self._page_hash(h, tokens, i)
            n = self.nodes.get(h)
            if n is None or n.page < 0 or not n.holds(at, tokens[i * P:(i + 1) * P]):
                break
            at = n
            pages.append(n.page)
        self.incref(pages)
        return pages, len(pages) * P

    def insert(self, tokens: list[int], pages: list[int]) -> None:
        P, h, at = self.page_size, 0, None
        full = min(len(tokens) // P, len(pages))
        if any(not 0 <= p < self.num_pages for p in pages[:full]):
            raise IndexError("page id out of range")
        for i in range(full):
            h = self._page_hash(h, tokens, i)
            n = self.nodes.get(h)
            if n is None:
                n = self.nodes[h] = _Node(at, h, list(tokens[i * P:(i + 1) * P]))
                if at is not None:
                    at.children += 1
            elif not n.holds(at, tokens[i * P:(i + 1) * P]):
                break  # other content with this hash
            at, p = n, pages[i]
            if n.page >= 0 or self.node_of[p]:
                continue
            n.page = p
            self.node_of[p] = n
        self._trim(at)

    def clear_cache(self) -> None:
        self.free.extend(self.lru)
        self.lru.clear()
        self.node_of = [None] * self.num_pages
        self.nodes.clear()

    def stats(self) -> dict:
        return {"num_pages": self.num_pages, "free": len(self.free), "cached": self.num_cached(), "evictable": len(self.lru)}
