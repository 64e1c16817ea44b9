"""Plain implementation of the step of sequences that share pages, from its definition, on lists."""

from kv4_ref import pages


class SharedPlan:
    def __init__(self, n_seq, page, width, n_pages):
        self.page, self.width, self.n_pages = page, width, n_pages
        self.lens = [0] * n_seq
        self.table = [[] for _ in range(n_seq)]

    def refs(self):
        count = [0] * self.n_pages
        for t in self.table:
            for p in t:
                count[p] += 1
        return count

    def step(self, grow, keep, parent, max_rows):
        """(starts, slots, positions), [(source, copy, kept rows)] and 0, or nothing changed and the
        error bits.  keep and parent may be None."""
        n, P = len(self.lens), self.page
        none = ([0] * (n + 1), [-1] * max_rows, [-1] * max_rows)
        parent = list(range(n)) if parent is None else parent
        err = 0
        for s in range(n):
            if not 0 <= parent[s] < n:
                err = 8
        if err:
            return none, [], err
        keep = [self.lens[p] for p in parent] if keep is None else keep
        for s in range(n):
            if keep[s] < 0 or keep[s] > self.lens[parent[s]] or grow[s] < 0 or \
                    keep[s] + grow[s] > self.width * P:
                err |= 8
        if sum(g for g in grow if g > 0) > max_rows and not err:
            err |= 32
        if err:
            return none, [], err
        table = [list(self.table[parent[s]][:pages(keep[s], P)]) for s in range(n)]
        holders = {}
        for s in range(n):
            for p in table[s]:
                holders.setdefault(p, []).append(s)
        writers = {}
        for s in range(n):
            if grow[s] and keep[s] % P:
                writers.setdefault(table[s][-1], []).append(s)
        free = [p for p in range(self.n_pages) if p not in holders]
        copies = []
        for s in range(n):
            if grow[s] and keep[s] % P:
                p = table[s][-1]
                if not (holders[p] == writers[p] and writers[p][0] == s):
                    if not free:
                        return none, [], 16
                    copies.append((p, free[0], keep[s] % P))
                    table[s][-1] = free.pop(0)
            for _ in range(pages(keep[s] + grow[s], P) - pages(keep[s], P)):
                if not free:
                    return none, [], 16
                table[s].append(free.pop(0))
        starts, slots, pos = [0], [], []
        for s in range(n):
            for r in range(keep[s], keep[s] + grow[s]):
                slots.append(table[s][r // P] * P + r % P)
                pos.append(r)
            starts.append(len(slots))
        self.table, self.lens = table, [k + g for k, g in zip(keep, grow)]
        pad = [-1] * (max_rows - len(slots))
        return (starts, slots + pad, pos + pad), copies, 0
