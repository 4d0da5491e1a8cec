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
