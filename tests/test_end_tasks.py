"""Stopping a node ends its background tasks, whatever they do with the first
cancellation."""
import asyncio

from crowdllama_amd.mesh.wire import end_tasks


def test_a_task_that_lost_a_cancellation_ends():
    async def go():
        lost = []

        async def loop():
            while True:
                try:
                    await asyncio.sleep(60)
                except asyncio.CancelledError:
                    if lost:
                        raise
                    lost.append(1)   # as wait_for does when it is done too

        async def fails():
            raise ValueError("ends by itself")

        tasks = [asyncio.create_task(loop()), asyncio.create_task(fails())]
        mine = list(tasks)
        await asyncio.sleep(0)
        await asyncio.wait_for(end_tasks(tasks), 10)
        assert lost and mine[0].cancelled() and mine[1].done() and not tasks
        await end_tasks(tasks)       # and none is none

    asyncio.run(go())


def test_a_task_may_take_its_time_to_clean_up():
    async def go():
        ended = []

        async def closes():
            try:
                await asyncio.sleep(60)
            finally:
                await asyncio.sleep(0.8)
                ended.append(1)

        tasks = [asyncio.create_task(closes())]
        await asyncio.sleep(0)
        await asyncio.wait_for(end_tasks(tasks), 10)
        assert ended

    asyncio.run(go())


def test_a_task_may_stop_the_node_that_it_belongs_to():
    async def go():
        tasks, closed = [], []

        async def stops():
            await end_tasks(tasks)
            closed.append(1)         # what a stop() does after that

        async def loop():
            await asyncio.sleep(60)

        tasks += [asyncio.create_task(loop()), asyncio.create_task(stops())]
        mine = list(tasks)
        await asyncio.wait(mine, timeout=10)
        assert closed and mine[0].cancelled() and not mine[1].cancelled()

    asyncio.run(go())
